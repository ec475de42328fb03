"""Operators around requests that share tokens of one KV pool, as cases that can be timed.

A program that serves many requests behind a common prompt (samples of one question, branches of a search, users of one
system prompt) keeps the prompt's K/V rows once: the request table of every such request names the same slots, and every slot
counts the requests that hold it.  Five kinds of calls: "decode" attends from one new token per request where groups of requests
share their first tokens, "prompt" is the step of prompts' chunks over the prefix that they share, "fork" gives new requests
another's tokens (the same slots, or copies of the rows in all layers), "free" lets go of requests' tokens, "compact" moves the slots
in use to the front of the pool.

listed() holds ordinary points of these kinds, draw() gives others of the same ranges.  Lengths come from the case alone,
values and slot numbers from the seed.  Where `own` is false, run() computes the plain forms: attention in float32, whole numbers and
rows as they are.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
PAD = 2147483647  # unused entries of the request table


def listed():
    return [
        # four samples of one question a few tokens in: the smallest decode step, where latency counts
        dict(name="decode_4_samples", kind="decode", batch=4, groups=1, alone=0, prefix_min=2011, prefix_max=2011, own_min=1, own_max=40,
             q_heads=32, kv_heads=8, head_dim=128, dtype="f16", lens=1),
        # a full batch of users behind one long system prompt
        dict(name="decode_64_one_prompt", kind="decode", batch=64, groups=1, alone=0, prefix_min=16384, prefix_max=16384, own_min=100,
             own_max=1500, q_heads=32, kv_heads=8, head_dim=128, dtype="f16", lens=2),
        # three ragged groups and a few requests on their own, MHA in bfloat16
        dict(name="decode_24_mha", kind="decode", batch=24, groups=3, alone=3, prefix_min=2500, prefix_max=9000, own_min=1, own_max=700,
             q_heads=32, kv_heads=32, head_dim=128, dtype="bf16", lens=3),
        # a large search over one document: many branches, few KV heads, 64-wide
        dict(name="decode_160_branches", kind="decode", batch=160, groups=2, alone=0, prefix_min=20000, prefix_max=32768, own_min=10,
             own_max=400, q_heads=28, kv_heads=4, head_dim=64, dtype="bf16", lens=4),
        # six short user turns behind one system prompt: the smallest prompt step
        dict(name="prompt_6_turns", kind="prompt", groups=1, rows_min=293, rows_max=293, prefix_min=6001, prefix_max=6001, q_heads=32,
             kv_heads=8, head_dim=128, dtype="f16", lens=5),
        # two groups of long user prompts, each behind a prefix of its own, bfloat16
        dict(name="prompt_2_groups_long", kind="prompt", groups=2, rows_min=3000, rows_max=5000, prefix_min=7000, prefix_max=9000, q_heads=32,
             kv_heads=8, head_dim=128, dtype="bf16", lens=6),
        # eight samples of one question are started, the question's slots shared
        dict(name="fork_8_samples", kind="fork", copies=False, parents=1, forks=8, len_min=2999, len_max=2999, slots=65536, layers=0, kv_heads=8,
             head_dim=128, dtype="f16", lens=7),
        # two requests that get copies of another's rows, all layers of a model
        dict(name="fork_2_copies", kind="fork", copies=True, parents=1, forks=2, len_min=6500, len_max=6500, slots=24000, layers=32, kv_heads=8,
             head_dim=128, dtype="f16", lens=9),
        # one request of a few tokens ends
        dict(name="free_1", kind="free", parents=1, forks=0, len_min=100, len_max=100, own_max=0, slots=65536, lens=10),
        # a search ends: branches of a few requests, and these
        dict(name="free_128_branches", kind="free", parents=8, forks=120, len_min=300, len_max=8000, own_max=600, slots=400000, lens=11),
        # a small 8-bit pool with little in use, here and there: the smallest call
        dict(name="compact_few_8bit", kind="compact", requests=3, len_min=50, len_max=500, slots=5000, layers=4, kv_heads=8, head_dim=128,
             dtype="e4m3", lens=12),
        # half of a pool is in use, here and there
        dict(name="compact_half", kind="compact", requests=24, len_min=200, len_max=2200, slots=60000, layers=12, kv_heads=8, head_dim=128,
             dtype="f16", lens=13),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _two(rng, lo, hi):
    return sorted((_log_int(rng, lo, hi), _log_int(rng, lo, hi)))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prompt", "fork", "free", "compact"])
    heads = [(32, 8), (32, 32), (8, 1), (16, 2), (28, 4)]
    while True:
        hq, hkv = rng.choice(heads)
        c = dict(kind=kind, lens=rng.randint(100, 10 ** 6))
        if kind in ("decode", "prompt"):
            low, high = _two(rng, 1, 32768)
            c.update(q_heads=hq, kv_heads=hkv, head_dim=rng.choice([128, 128, 128, 64]), dtype=rng.choice(["f16", "bf16"]),
                     groups=_log_int(rng, 1, 12), prefix_min=low, prefix_max=high)
        if kind == "decode":
            low, high = _two(rng, 1, 3000)
            batch = _log_int(rng, 1, 160)
            c.update(batch=batch, groups=min(c["groups"], batch), own_min=low, own_max=high)
            c.update(alone=rng.choice([0, 0, rng.randint(0, batch - c["groups"])]))
        elif kind == "prompt":
            low, high = _two(rng, 1, 8192)
            c.update(rows_min=low, rows_max=high)
        else:
            c.update(slots=_log_int(rng, 300, 400000))
            low, high = _two(rng, 1, 16384)
            if kind == "compact":
                c.update(requests=_log_int(rng, 1, 200), len_min=low, len_max=high)
            else:
                c.update(parents=_log_int(rng, 1, 20), forks=_log_int(rng, 1, 200), len_min=low, len_max=high)
            if kind == "free":
                c.update(own_max=rng.choice([0, _log_int(rng, 1, 1000)]))
            else:
                c.update(kv_heads=hkv, head_dim=rng.choice([128, 64]), dtype=rng.choice(["f16", "bf16", "e4m3"]), layers=_log_int(rng, 1, 32))
            if kind == "fork":
                c.update(copies=rng.random() < 0.5)
                c.update(layers=c["layers"] if c["copies"] else 0)
        w, most = work(c), [work(d) for d in listed() if d["kind"] == kind]
        if w["bytes"] > max(m["bytes"] for m in most) or w["flops"] > max(m["flops"] for m in most) or _room(c) > 3.3e9 or not _fits(c):
            continue
        return c


def _room(c):
    """Elements of the pool, or of what the plain form holds at once."""
    if c["kind"] == "decode":
        pre, size, own_len = _decode_shape(c)
        rows = len(pre) * max(pre) + c["batch"] * max(own_len)
        return 3 * rows * 2 * c["kv_heads"] * c["head_dim"] + 4 * c["q_heads"] * (len(pre) * max(size) * max(pre) + c["batch"] * max(own_len))
    if c["kind"] == "prompt":
        pre, rows = _prompt_shape(c)
        return 3 * len(pre) * max(pre) * 2 * c["kv_heads"] * c["head_dim"] // 2 + 2 * len(pre) * max(rows) * c["q_heads"] * max(pre) // 2
    if c["kind"] == "free":
        return c["slots"]
    return c["slots"] * max(1, c["layers"]) * 2 * c["kv_heads"] * c["head_dim"]


def _fits(c):
    """Whether the slots that the case needs are there."""
    if c["kind"] == "fork":
        pl, fl = _fork_shape(c)
        return sum(pl) + (sum(fl) if c["copies"] else 0) <= c["slots"]
    if c["kind"] == "free":
        pl, _, ol = _free_shape(c)
        return sum(pl) + sum(ol) <= c["slots"]
    if c["kind"] == "compact":
        return sum(_compact_shape(c)) <= c["slots"]
    return True


# ------------------------------------------------------------------------------------------------ the cases' lengths
def _ends(r, n, low, high):
    """n numbers between low and high, both among them where there are two."""
    x = [r.randint(low, high) for _ in range(n)]
    if n:
        x[-1] = low
        x[0] = high
    return x


def _decode_shape(c):
    """(prefixes, sizes of the groups, own tokens of the requests)."""
    r = random.Random(c["lens"])
    pre = _ends(r, c["groups"], c["prefix_min"], c["prefix_max"])
    cuts = sorted(r.sample(range(1, c["batch"] - c["alone"]), c["groups"] - 1)) if c["groups"] > 1 else []
    size = [b - a for a, b in zip([0] + cuts, cuts + [c["batch"] - c["alone"]])]
    return pre, size, _ends(r, c["batch"], c["own_min"], c["own_max"])


def _prompt_shape(c):
    r = random.Random(c["lens"])
    return _ends(r, c["groups"], c["prefix_min"], c["prefix_max"]), _ends(r, c["groups"], c["rows_min"], c["rows_max"])


def _fork_shape(c):
    """(lengths of the parents, lengths of the forks: fork i is one of parent i * parents // forks)."""
    r = random.Random(c["lens"])
    pl = _ends(r, c["parents"], c["len_min"], c["len_max"])
    own_part = r.random() < 0.5  # a fork has all of its parent's tokens, or some first ones
    fl = [pl[i * c["parents"] // c["forks"]] for i in range(c["forks"])]
    return pl, [r.randint(1, n) for n in fl] if own_part else fl


def _free_shape(c):
    """(lengths of the parents, shared tokens of the forks, own tokens of the forks)."""
    r = random.Random(c["lens"])
    pl = _ends(r, c["parents"], c["len_min"], c["len_max"])
    return pl, [r.randint(1, pl[i % c["parents"]]) for i in range(c["forks"])], [r.randint(0, c["own_max"]) for _ in range(c["forks"])]


def _compact_shape(c):
    return _ends(random.Random(c["lens"]), c["requests"], c["len_min"], c["len_max"])


def _row_bytes(c):
    return 2 * c["kv_heads"] * (c["head_dim"] + 1 if c["dtype"] == "e4m3" else 2 * c["head_dim"])


def work(case):
    c = case
    if c["kind"] == "decode":
        pre, size, own_len = _decode_shape(c)
        d, hq, row = c["head_dim"], c["q_heads"], 2 * c["kv_heads"] * c["head_dim"] * 2 + 4
        pairs = sum(p * n for p, n in zip(pre, size)) + sum(own_len)
        return {"bytes": (sum(pre) + sum(own_len)) * row + c["batch"] * hq * (4 * d + 4), "flops": 4 * d * hq * pairs}
    if c["kind"] == "prompt":
        pre, rows = _prompt_shape(c)
        d, hq, row = c["head_dim"], c["q_heads"], 2 * c["kv_heads"] * c["head_dim"] * 2 + 4
        return {"bytes": sum(pre) * row + sum(rows) * hq * (4 * d + 8), "flops": 4 * d * hq * sum(p * n for p, n in zip(pre, rows))}
    if c["kind"] == "fork":
        pl, fl = _fork_shape(c)
        read = max(fl) if c["parents"] == 1 else sum(pl)
        if c["copies"]:
            return {"bytes": 2 * sum(fl) * c["layers"] * _row_bytes(c) + sum(fl) * 12 + 4 * read, "flops": 0}
        return {"bytes": 4 * sum(fl) + 4 * read + 8 * read, "flops": 0}
    if c["kind"] == "free":
        pl, shared, own_len = _free_shape(c)
        return {"bytes": 4 * (sum(pl) + sum(shared) + sum(own_len)) + 8 * (sum(pl) + sum(own_len)), "flops": 0}
    n = sum(_compact_shape(c))
    moved = n * (c["slots"] - n) // c["slots"]  # used slots past the number in use, where they lie anywhere
    return {"bytes": 2 * moved * c["layers"] * _row_bytes(c) + 8 * c["slots"] + 8 * n, "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs
def _rows(g, shape, kv_heads, dtype):
    """K heads then V heads: K with a few strong channels, V of a size that differs from token to token."""
    x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)
    channel = torch.rand(kv_heads, shape[-1], generator=g, device=DEV)
    x[..., :kv_heads, :] *= 0.5 + 2.5 * (channel > 0.95)
    x[..., kv_heads:, :] *= torch.exp(0.5 * torch.randn(*shape[:-2], 1, 1, generator=g, device=DEV))
    return x.to(dtype)


def _pool(g, slots, c, layers=None):
    """[slots, 2 kv_heads, head_dim], or with `layers` in front, filled some rows at a time."""
    total = slots * (layers or 1)
    pool = torch.empty(total, 2 * c["kv_heads"], c["head_dim"], dtype=DTYPES[c["dtype"]], device=DEV)
    step = max(1, (1 << 28) // (2 * c["kv_heads"] * c["head_dim"]))
    for i in range(0, total, step):
        n = min(step, total - i)
        pool[i:i + n] = _rows(g, (n, 2 * c["kv_heads"], c["head_dim"]), c["kv_heads"], DTYPES[c["dtype"]])
    return pool.view(layers, slots, 2 * c["kv_heads"], c["head_dim"]) if layers else pool


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def _starts(lens):
    return _ints([sum(lens[:b]) for b in range(len(lens))])


def _tables(g, rows, longest):
    return torch.full((rows + 3, longest + 5), PAD, dtype=torch.int32, device=DEV), torch.randperm(rows + 3, generator=g, device=DEV)[:rows].to(torch.int32)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    return dict(case=c, **{"decode": _prepare_decode, "prompt": _prepare_prompt, "fork": _prepare_fork, "free": _prepare_free,
                           "compact": _prepare_compact}[c["kind"]](c, g))


def _prepare_decode(c, g):
    pre, size, own_len = _decode_shape(c)
    shared = [p for p, n in zip(pre, size) for _ in range(n)] + [0] * c["alone"]
    lens = [p + n for p, n in zip(shared, own_len)]
    slots = sum(pre) + sum(own_len) + 50
    table, req = _tables(g, c["batch"], max(lens))
    slot = torch.randperm(slots, generator=g, device=DEV).to(torch.int32)
    at = b = 0
    starts = []
    for p, n in zip(pre, size):
        starts.append(b)
        table[req[b:b + n].long(), :p] = slot[at:at + p]
        at, b = at + p, b + n
    for b, n in enumerate(own_len):
        table[int(req[b]), shared[b]:shared[b] + n] = slot[at:at + n]
        at += n
    return dict(pool=_pool(g, slots, c), table=table, req=req, len=_ints(lens), longest=max(lens), g_start=_ints(starts), g_size=_ints(size),
                g_req=req[_ints(starts).long()].contiguous(), g_prefix=_ints(pre), longest_prefix=max(pre), longest_own=max(own_len),
                q=torch.randn(c["batch"], c["q_heads"], c["head_dim"], generator=g, device=DEV).to(DTYPES[c["dtype"]]),
                shape=(max(size), max(own_len)))


def _prepare_prompt(c, g):
    pre, rows = _prompt_shape(c)
    slots = sum(pre) + 50
    table, req = _tables(g, c["groups"], max(pre))
    slot = torch.randperm(slots, generator=g, device=DEV).to(torch.int32)
    for i, p in enumerate(pre):
        table[int(req[i]), :p] = slot[sum(pre[:i]):sum(pre[:i]) + p]
    q = torch.randn(sum(rows), c["q_heads"], c["head_dim"], generator=g, device=DEV).to(DTYPES[c["dtype"]])
    return dict(pool=_pool(g, slots, c), table=table, g_start=_starts(rows), g_size=_ints(rows), g_req=req, g_prefix=_ints(pre), longest_prefix=max(pre),
                longest_rows=max(rows), q=q, o=torch.zeros_like(q), m=torch.empty(q.shape[:2], device=DEV), l=torch.empty(q.shape[:2], device=DEV))


def _prepare_fork(c, g):
    pl, fl = _fork_shape(c)
    table, req = _tables(g, c["parents"] + c["forks"], max(pl))
    slot = torch.randperm(c["slots"], generator=g, device=DEV)
    mem = torch.zeros(c["slots"], dtype=torch.int32, device=DEV)
    mem[slot[:sum(pl)]] = 1
    for i, n in enumerate(pl):
        table[int(req[i]), :n] = slot[sum(pl[:i]):sum(pl[:i]) + n].to(torch.int32)
    parent = [i * c["parents"] // c["forks"] for i in range(c["forks"])]
    s = dict(table=table, mem=mem, src=req[_ints(parent).long()].contiguous(), dst=req[c["parents"]:].contiguous(), len=_ints(fl), longest=max(fl))
    if c["copies"]:
        s.update(index=slot[sum(pl):sum(pl) + sum(fl)].contiguous(), start=_starts(fl), pool=_pool(g, c["slots"], c, c["layers"]), scales=None)
        if c["dtype"] == "e4m3":
            s["scales"] = torch.randint(100, 150, (c["layers"], c["slots"], 2 * c["kv_heads"]), dtype=torch.uint8, generator=g, device=DEV)
    return s


def _prepare_free(c, g):
    pl, shared, own_len = _free_shape(c)
    lens = pl + [a + b for a, b in zip(shared, own_len)]
    table, req = _tables(g, len(lens), max(lens))
    slot = torch.randperm(c["slots"], generator=g, device=DEV).to(torch.int32)
    mem = torch.randint(0, 2, (c["slots"],), dtype=torch.int32, generator=g, device=DEV)  # (others' slots)
    at = 0
    mem[slot[:sum(pl) + sum(own_len)].long()] = 0
    for i, n in enumerate(pl):
        table[int(req[i]), :n] = slot[at:at + n]
        mem[slot[at:at + n].long()] += 1
        at += n
    for i, (a, b) in enumerate(zip(shared, own_len)):
        row, parent = int(req[len(pl) + i]), int(req[i % len(pl)])
        table[row, :a] = table[parent, :a]
        mem[table[parent, :a].long()] += 1
        table[row, a:a + b] = slot[at:at + b]
        mem[slot[at:at + b].long()] = 1
        at += b
    return dict(table=table, req=req, len=_ints(lens), longest=max(lens), mem=mem.clone(), mem_before=mem)


def _prepare_compact(c, g):
    lens = _compact_shape(c)
    table, req = _tables(g, len(lens), max(lens))
    slot = torch.randperm(c["slots"], generator=g, device=DEV).to(torch.int32)
    mem = torch.zeros(c["slots"], dtype=torch.int32, device=DEV)
    for i, n in enumerate(lens):
        table[int(req[i]), :n] = slot[sum(lens[:i]):sum(lens[:i]) + n]
    mem[slot[:sum(lens)].long()] = 1 + torch.randint(0, 2, (sum(lens),), dtype=torch.int32, generator=g, device=DEV)
    scales = None
    if c["dtype"] == "e4m3":
        scales = torch.randint(100, 150, (c["layers"], c["slots"], 2 * c["kv_heads"]), dtype=torch.uint8, generator=g, device=DEV)
    return dict(table=table.clone(), table_before=table, req=req, len=_ints(lens), longest=max(lens), mem=mem.clone(), mem_before=mem,
                pool=_pool(g, c["slots"], c, c["layers"]), scales=scales)


# ------------------------------------------------------------------------------------------------ plain forms
def _prefix_rows(c, s):
    """(K [groups, kv_heads, head_dim, tokens], V [groups, kv_heads, tokens, head_dim], which tokens exist [groups, tokens]) of the shared prefixes."""
    at = torch.arange(s["longest_prefix"], device=DEV)[None]
    there = at < s["g_prefix"][:, None]
    slots = torch.where(there, s["table"][s["g_req"].long(), :s["longest_prefix"]], 0).long()
    rows = s["pool"][slots].float()
    hkv = c["kv_heads"]
    return rows[:, :, :hkv].permute(0, 2, 3, 1).contiguous(), rows[:, :, hkv:].permute(0, 2, 1, 3).contiguous(), there


def _group_rows(c, s, rows, most):
    """Rows of q by group: [groups, most, kv_heads, heads of a KV head, head_dim], their numbers and whether each exists."""
    i = torch.arange(most, device=DEV)[None]
    there = i < s["g_size"][:, None]
    at = torch.where(there, s["g_start"][:, None] + i, 0).long()
    return rows[at], at, there


def _decode(c, s):
    hkv, hq, d = c["kv_heads"], c["q_heads"], c["head_dim"]
    group, most, own_most = hq // hkv, *s["shape"]
    q = s["q"].float().view(c["batch"], hkv, group, d)
    k, v, there = _prefix_rows(c, s)
    qg, at, row_there = _group_rows(c, s, q, most)
    n = len(k)
    x = qg.permute(0, 2, 1, 3, 4).reshape(n, hkv, most * group, d).matmul(k) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~there[:, None, None], -math.inf)
    # own tokens of every request, behind its group's prefix
    first = torch.zeros_like(s["len"])
    first[at[row_there]] = s["g_prefix"][:, None].expand(-1, most)[row_there]
    pos = first[:, None] + torch.arange(own_most, device=DEV)[None]
    own_there = pos < s["len"][:, None]
    slots = torch.where(own_there, s["table"][s["req"].long()].gather(1, pos.clamp(max=s["longest"] - 1).long()), 0).long()
    rows = s["pool"][slots].float()
    y = q.matmul(rows[:, :, :hkv].permute(0, 2, 3, 1).contiguous()) * (1.0 / math.sqrt(d))
    y = y.masked_fill(~own_there[:, None, None], -math.inf)
    v_own = rows[:, :, hkv:].permute(0, 2, 1, 3).contiguous()
    del rows
    x = x.view(n, hkv, most, group, -1)
    m = y.amax(-1)
    m[at[row_there]] = torch.maximum(m[at[row_there]], x.amax(-1).permute(0, 2, 1, 3)[row_there])
    x = torch.exp(x - m[at].permute(0, 2, 1, 3)[..., None])
    y = torch.exp(y - m[..., None])
    l, o = y.sum(-1), y.matmul(v_own)
    l[at[row_there]] += x.sum(-1).permute(0, 2, 1, 3)[row_there]
    far = x.view(n, hkv, most * group, -1).matmul(v).view(n, hkv, most, group, d)
    o[at[row_there]] += far.permute(0, 2, 1, 3, 4)[row_there]
    o = o / l[..., None]
    return o.reshape(s["q"].shape).to(s["q"].dtype), (m + torch.log(l)).reshape(c["batch"], hq)


def _prompt(c, s):
    hkv, hq, d = c["kv_heads"], c["q_heads"], c["head_dim"]
    group, most = hq // hkv, s["longest_rows"]
    k, v, there = _prefix_rows(c, s)
    qg, at, row_there = _group_rows(c, s, s["q"].float().view(-1, hkv, group, d), most)
    n = len(k)
    x = qg.permute(0, 2, 1, 3, 4).reshape(n, hkv, most * group, d).matmul(k).mul_(1.0 / math.sqrt(d))
    x.masked_fill_(~there[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    o = (x.matmul(v) / l).view(n, hkv, most, group, d).permute(0, 2, 1, 3, 4)
    lse = (m + torch.log(l)).view(n, hkv, most, group).permute(0, 2, 1, 3)
    s["o"][at[row_there]] = o[row_there].reshape(-1, hq, d).to(s["o"].dtype)
    return s["o"], lse[row_there].reshape(-1, hq)


def _fork(c, s):
    at = torch.arange(s["longest"], device=DEV)[None]
    there = at < s["len"][:, None]
    row, col = there.nonzero(as_tuple=True)
    slots = s["table"][s["src"].long()[row], col]
    if not c["copies"]:
        s["table"][s["dst"].long()[row], col] = slots
        s["mem"].index_add_(0, slots.long(), torch.ones_like(slots))
        return s["table"], s["mem"]
    index = s["index"][s["start"].long()[row] + col]
    s["table"][s["dst"].long()[row], col] = index.to(torch.int32)
    raw = s["pool"].view(torch.int64)  # (rows as bits, eight bytes at a time)
    raw[:, index] = raw[:, slots.long()]
    if s["scales"] is not None:
        s["scales"][:, index] = s["scales"][:, slots.long()]
    return s["table"], s["pool"], s["scales"]


def _free(c, s):
    at = torch.arange(s["longest"], device=DEV)[None]
    slots = s["table"][s["req"].long(), :s["longest"]][at < s["len"][:, None]]
    before = (s["mem"] > 0).sum()
    s["mem"].index_add_(0, slots.long(), torch.full_like(slots, -1))
    return s["mem"], int(before - (s["mem"] > 0).sum())


def _compact(c, s):
    used = s["mem"] > 0
    count = int(used.sum())
    source, hole = used[count:].nonzero().squeeze(1) + count, (~used[:count]).nonzero().squeeze(1)
    remap = torch.where(used, torch.arange(c["slots"], device=DEV), -1).to(torch.int32)
    remap[source] = hole.to(torch.int32)
    raw = s["pool"].view(torch.int64)  # (rows as bits, eight bytes at a time)
    raw[:, hole] = raw[:, source]
    if s["scales"] is not None:
        s["scales"][:, hole] = s["scales"][:, source]
    s["mem"][hole] = s["mem"][source]
    s["mem"][source] = 0
    at = torch.arange(s["longest"], device=DEV)[None]
    row, col = (at < s["len"][:, None]).nonzero(as_tuple=True)
    row = s["req"].long()[row]
    s["table"][row, col] = remap[s["table"][row, col].long()]
    return remap, s["mem"], s["table"], s["pool"], s["scales"]


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "free":  # (the counts as they are before the call)
        s["mem"].copy_(s["mem_before"])
    if c["kind"] == "compact":  # (rows that a pass has moved lie where they were, too)
        s["mem"].copy_(s["mem_before"])
        s["table"].copy_(s["table_before"])
    if own:
        import loongserve_amd as lsa
        if c["kind"] == "decode":
            hkv = c["kv_heads"]
            return lsa.longserve_shared_prefix_decode_attention(s["q"], s["table"], s["req"], s["len"], s["longest"], s["pool"][:, :hkv], s["pool"][:, hkv:],
                                                                s["g_start"], s["g_size"], s["g_req"], s["g_prefix"], s["longest_prefix"],
                                                                max_own_len=s["longest_own"])
        if c["kind"] == "prompt":
            hkv = c["kv_heads"]
            s["m"].fill_(-math.inf)
            s["l"].zero_()
            lsa.shared_prefix_attention_fwd(s["q"], s["pool"][:, :hkv], s["pool"][:, hkv:], s["o"], s["g_start"], s["g_size"], s["table"], s["g_req"],
                                            s["g_prefix"], s["longest_rows"], s["longest_prefix"], s["m"], s["l"])
            return s["o"], torch.log2(s["l"]).add_(s["m"]).mul_(math.log(2.0))
        if c["kind"] == "fork":
            if not c["copies"]:
                lsa.fork_requests(s["table"], s["src"], s["dst"], s["len"], s["longest"], s["mem"])
                return s["table"], s["mem"]
            lsa.copy_requests(s["table"], s["src"], s["dst"], s["len"], s["start"], s["longest"], s["index"], s["pool"], s["scales"])
            return s["table"], s["pool"], s["scales"]
        if c["kind"] == "free":
            return s["mem"], lsa.release_requests(s["table"], s["req"], s["len"], s["longest"], s["mem"])
        remap = lsa.compact_pool(s["mem"], s["pool"], s["table"], s["req"], s["len"], s["longest"], s["scales"])
        return remap, s["mem"], s["table"], s["pool"], s["scales"]
    return {"decode": _decode, "prompt": _prompt, "fork": _fork, "free": _free, "compact": _compact}[c["kind"]](c, s)


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    """The definitions of the attention operators in float64, KV head by KV head; the others return whole numbers and rows as they were."""
    c = case
    if c["kind"] not in ("decode", "prompt") or work(c)["flops"] > 4e12:
        return None
    s = prepare(case, seed)
    hkv, d = c["kv_heads"], c["head_dim"]
    group = c["q_heads"] // hkv
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)

    def attend(rows, slots):
        for h in range(hkv):
            k, v = s["pool"][slots, h].double(), s["pool"][slots, hkv + h].double()
            heads = slice(h * group, (h + 1) * group)
            x = (s["q"][rows, heads].double().reshape(-1, d) @ k.T) / math.sqrt(d)
            top = torch.logsumexp(x, -1)
            o[rows, heads] = (torch.exp(x - top[:, None]) @ v).view(-1, group, d)
            lse[rows, heads] = top.view(-1, group)

    if c["kind"] == "decode":
        for b, n in enumerate(s["len"].tolist()):
            attend(slice(b, b + 1), s["table"][int(s["req"][b]), :n].long())
        return o, lse
    for i, (at, n) in enumerate(zip(s["g_start"].tolist(), s["g_size"].tolist())):
        slots = s["table"][int(s["g_req"][i]), :int(s["g_prefix"][i])].long()
        for r in range(at, at + n, 1024):
            attend(slice(r, min(at + n, r + 1024)), slots)
    return o, lse
