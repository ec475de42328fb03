"""Decode over the 8-bit pool where its exponents are at their ends: slots that nobody wrote, V rows of zeros, very small and very large ones."""
import math

import numpy as np
import pytest
import torch

from oracle import pool8_oracle as orc
from tests.test_gpu_pool8 import PAD, Case

K8 = ["e4m3-f16", "e4m3-bf16"]


class Unwritten(Case):
    """A Case whose slots that no request holds, slot 0 among them, have the exponent byte 255 (E8M0's NaN) beside their NaN rows."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        n = self.values.shape[0]
        used = torch.zeros(n, dtype=torch.bool)
        used[self.table[(self.table >= 0) & (self.table < n)].long()] = True
        if used[0]:
            to = int((~used).nonzero()[0])
            self.table[self.table == 0] = to
            used[0], used[to] = False, True
            for t in (self.values, self.pool.view(torch.uint8), self.scales):
                t[[0, to]] = t[[to, 0]]
        self.scales[(~used).cuda()] = 255
        assert not used[0] and not (self.table == 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", K8)
@pytest.mark.parametrize("lens,holes", [([1, 33, 700, 0, 64], []), ([70, 40], [(0, 0), (0, 33), (0, 34), (1, 39)]),
                                        ([9000, 3], [(0, 0), (0, 8999), (0, 4000), (1, 1)]), ([96, 96, 96], [])])
def test_exponents_of_slots_that_are_not_seen_do_not_matter(lsa, kind, lens, holes):
    """Slots are neutral where a position does not exist (past a request's end, a hole of the table), whatever slot 0 holds; in both launch forms."""
    c = Unwritten(kind, len(lens), 8, 2, 128, lens, seed=21, holes=holes)
    for max_len in (None, 1 << 17):
        c.check(c.run(lsa, max_len=max_len))
        c.check(c.run(lsa, 50, 3, max_len=max_len), 50, 3)


def _rows_at(exponents, D, seed):
    """(bytes of e4m3 values, exponent bytes, float64 values) of rows [tokens, heads] with the largest element in (224, 448] * 2^e; e = None: zeros."""
    g = torch.Generator().manual_seed(seed)
    T, H = len(exponents), len(exponents[0])
    x = torch.randn(T, H, D, generator=g, dtype=torch.float64)
    q = orc.round_e4m3(x / x.abs().amax(-1, keepdim=True) * 440)
    e = torch.tensor([[-126 if y is None else y for y in row] for row in exponents])
    q[torch.tensor([[y is None for y in row] for row in exponents])] = 0
    return q.float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8), q * torch.pow(2.0, e.double())[..., None], e


class Ends:
    """One request whose V rows have the exponents given (per token and KV head), K ordinary; `lift` names tokens whose scores lie that many
    nats above (or below) what the others have."""

    def __init__(self, dtype, exponents, lift=(), Hq=8, Hkv=2, D=128, seed=0):
        T = len(exponents)
        g = torch.Generator().manual_seed(seed)
        base = torch.randn(Hkv, D, generator=g, dtype=torch.float64)
        self.q = (base.repeat_interleave(Hq // Hkv, 0) + 0.1 * torch.randn(Hq, D, generator=g, dtype=torch.float64))[None].to(dtype)
        k = torch.randn(T, Hkv, D, generator=g, dtype=torch.float64)
        for t, nats in lift:
            k[t] = base * (nats * math.sqrt(D) / (base * base).sum(-1, keepdim=True))
        kq, ke = orc.quantise(k)
        v8, vb, v, self.e = _rows_at(exponents, D, seed + 1)
        self.k, self.v, self.T, self.Hkv, self.Hq, self.D = kq * torch.pow(2.0, (ke - 127).double())[..., None], v, T, Hkv, Hq, D
        order = torch.randperm(T + 3, generator=g)[:T]
        pool = torch.full((T + 3, 2 * Hkv, D), 0x7F, dtype=torch.uint8)
        scales = torch.full((T + 3, 2 * Hkv), 255, dtype=torch.uint8)
        pool[order] = torch.cat([kq.float().to(torch.float8_e4m3fn).view(torch.uint8), v8.view(torch.uint8)], 1)
        scales[order] = torch.cat([ke.to(torch.uint8), vb], 1)
        self.pool, self.scales, self.table = pool.cuda().view(torch.float8_e4m3fn), scales.cuda(), order.to(torch.int32)[None].cuda()

    def check(self, lsa, max_len=None):
        T, h, D = self.T, self.Hkv, self.D
        i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        o, l = lsa.longserve_fp8_decode_attention(self.q.cuda(), self.table, i(0), i(T), T if max_len is None else max_len, self.pool[:, :h], self.pool[:, h:],
                                                  self.scales[:, :h], self.scales[:, h:])
        G = self.Hq // h
        q, k, v = self.q[0].double(), self.k.repeat_interleave(G, 1), self.v.repeat_interleave(G, 1)
        s = torch.einsum("hd,nhd->hn", q, k) / math.sqrt(D)
        size = torch.einsum("hd,nhd->hn", q.abs(), k.abs()).amax(-1) / math.sqrt(D)
        lse = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[:, None])
        want, mean = torch.einsum("hn,nhd->hd", p, v), torch.einsum("hn,nhd->hd", p, v.abs())
        # float32 (eps = 2^-24, half a step): a score is a sum of D products, twice (numerator and sum); up to 30 eps for each exponential, whose argument is
        # up to some 24 where the weight counts, its division and the parts of the weight (2^-22 = 4 eps); sums in blocks of 32 tokens.  A weight is kept to
        # 2^-25 beside a largest one of 2^7 at least, and stands for e4m3 values of up to 448 * 2^e.  Results below 2^-126 may be flushed.
        eps = 2.0 ** -24
        rel = 2 * ((D + 8) * eps * size + 30 * eps + (T / 32 + 40) * eps)
        top = (p * torch.pow(2.0, self.e.double()).repeat_interleave(G, 1).T).amax(-1)
        tol = rel[:, None] * mean + (T * 2.0 ** -32 * 448 * top)[:, None] + 2.0 ** -126
        got = o[0].cpu().double()
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()
        assert ((l[0].cpu().double() - lse).abs() <= rel + 8 * eps * lse.abs()).all(), (l[0].cpu().double() - lse).abs().max()


def _ends(name, T):
    """Exponents of T tokens, and tokens with scores of their own."""
    r = torch.Generator().manual_seed(5)
    pick = lambda *v: [[v[int(x)] for x in row] for row in torch.randint(0, len(v), (T, 2), generator=r)]  # noqa: E731
    if name == "a zero row takes the weight":
        return [[None, None]] + pick(-7, -8)[1:], [(0, 15.0)]
    if name == "zero rows":
        return pick(None), []
    if name == "zero rows beside ordinary ones":
        return pick(None, -7, -8), []
    if name == "very small rows beside ordinary ones":
        return pick(-100, -7), [(T // 2, 12.0)]
    if name == "zero rows beside 2^61 and more":
        return pick(None, 54, 61), []
    if name == "small rows that take the weight beside the largest there are":
        return pick(-110, -100)[:-1] + [[118, 118]], [(T - 1, -60.0), (0, 5.0)]
    if name == "the largest there are":
        return pick(112, 118), []
    if name == "the smallest there are":
        return pick(-126, -124), []
    if name == "all sizes":
        return pick(None, -126, -100, -80, -60, -30, 0, 30, 60, 90, 110), []
    assert name == "growing from the smallest to the largest"
    return [[-126 + 240 * t // T, 114 - 240 * t // T] for t in range(T)], []


NAMES = ["a zero row takes the weight", "zero rows", "zero rows beside ordinary ones", "very small rows beside ordinary ones", "zero rows beside 2^61 and more",
         "small rows that take the weight beside the largest there are", "the largest there are", "the smallest there are", "all sizes",
         "growing from the smallest to the largest"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("T,max_len", [(333, None), (333, 1 << 17), (4100, None)])
def test_v_rows_of_any_exponents(lsa, dtype, name, T, max_len):
    """Both launch forms, exponents from -126 to 118."""
    exponents, lift = _ends(name, T)
    Ends(dtype, exponents, lift, seed=T).check(lsa, max_len)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "e4m3-f16"])
def test_lengths_and_windows_as_numpy_integers(lsa, kind):
    """What a scheduler that keeps its lengths in numpy passes."""
    c = Case(kind, 2, 8, 2, 128, [70, 31], seed=24)
    for window, sinks in ((50, 3), (None, 0)):
        got = c.run(lsa, window if window is None else np.int64(window), np.int32(sinks), max_len=np.int64(70))
        c.check(got, window, sinks)
    if c.k8:
        i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        a = (c.pool, c.scales, c.table.cuda(), c.req.cuda(), c.len.cuda(), i(0, 70))
        outs = [torch.zeros(101, 4, 128, dtype=torch.float16, device="cuda") for _ in range(2)]
        lsa.kv_gather_fp8(*a, 70, outs[0])
        lsa.kv_gather_fp8(*a, np.int64(70), outs[1])
        assert torch.equal(*outs) and outs[0].any()
    with pytest.raises(ValueError, match="window"):
        c.run(lsa, np.int64(0), 2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", K8)
@pytest.mark.parametrize("lens", [[300, 31], [9000]])
def test_exponents_as_e8m0(lsa, kind, lens):
    """The exponent bytes as a float8_e8m0fnu tensor: written, read back and attended over as the same bytes of uint8 are."""
    c = Case(kind, len(lens), 8, 2, 128, lens, seed=23)
    e8 = torch.float8_e8m0fnu
    want = c.run(lsa)
    c.scales = c.scales.view(e8)
    got = c.run(lsa)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    x = torch.randn(7, 4, 128, generator=torch.Generator().manual_seed(1)).to(c.dtype).cuda()
    idx = torch.arange(7, device="cuda")
    outs = []
    for t in (torch.uint8, e8):
        pool, sc = torch.zeros(9, 4, 128, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.zeros(9, 4, dtype=torch.uint8, device="cuda")
        lsa.kv_scatter_fp8(x, idx, pool, sc.view(t))
        out = torch.zeros(7, 4, 128, dtype=c.dtype, device="cuda")
        i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        lsa.kv_gather_fp8(pool, sc.view(t), idx.int().view(1, 7), i(0), i(7), i(0), 7, out)
        outs.append((pool.view(torch.uint8), sc, out))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [70, 3001])
def test_rows_move_with_their_exponents(lsa, n):
    """The decoding-stage migration, the context migration and kv_scatter on a pool in 8 bits: rows and, in a second call, exponents; decode gives
    the same bits from the new slots."""
    L, H, Hq, D, slots = 2, 8, 16, 128, 4000
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator().manual_seed(n)
    rows = torch.randn(L, n, 2 * H, D, generator=g) * torch.exp(3 * torch.randn(L, n, 2 * H, 1, generator=g))
    mem, there = (lsa.LongServeMemoryManager(slots, torch.float8_e4m3fn, H, D, L) for _ in range(2))
    at = torch.randperm(slots, generator=g)[:n].cuda()
    for layer in range(L):
        lsa.kv_scatter_fp8(rows[layer].half().cuda(), at, mem.kv_buffer[layer], mem.kv_scales[layer])
    q = torch.randn(1, Hq, D, generator=g).half().cuda()
    table = torch.full((3, n + 7), PAD, dtype=torch.int32, device="cuda")
    table[1, :n] = at.int()

    def decode(pool, scales, t):
        return lsa.longserve_fp8_decode_attention(q, t, i(1), i(n), n, pool[:, :H], pool[:, H:], scales[:, :H], scales[:, H:])
    want = [decode(mem.kv_buffer[layer], mem.kv_scales[layer], table) for layer in range(L)]

    def same(pool, scales, t):
        for layer in range(L):
            # (as bits: a row past fp16 is infinite, so NaN in the pool)
            assert all(torch.equal(x.view(torch.int32), y.view(torch.int32)) for x, y in zip(decode(pool[layer], scales[layer], t), want[layer]))
    # the decoding-stage migration of the whole context
    to = torch.randperm(slots, generator=g)[:n].to(torch.int32).cuda()
    state, new = torch.ones(slots, dtype=torch.int32, device="cuda"), torch.full_like(table, PAD)
    for src, dst in ((mem.kv_buffer, there.kv_buffer), (mem.kv_scales[..., None], there.kv_scales[..., None])):
        buf = torch.zeros((L, n, *src.shape[2:]), dtype=torch.uint8, device="cuda").view(src.dtype)
        lsa.decoding_stage_migration_sender_kernel(buf, table, state, src, i(1), i(n), i(n))
        lsa.decoding_stage_migration_receiver_kernel(buf, new, dst, to, i(1), i(n), i(0))
    assert torch.equal(new[1, :n], to) and int((state == 0).sum()) == n
    same(there.kv_buffer, there.kv_scales, new)
    # packed rows copied into their slots and registered; and row by row, from one slot to another
    for how in ("register", "scatter"):
        pool, scales = torch.zeros_like(there.kv_buffer.view(torch.uint8)), torch.zeros_like(there.kv_scales)
        new = torch.full_like(table, PAD)
        for layer in range(L):
            for k, (src, dst) in enumerate(((mem.kv_buffer.view(torch.uint8)[layer], pool[layer]), (mem.kv_scales[layer], scales[layer]))):
                if how == "register":
                    lsa.destindex_copy_and_register_kv(1, i(n), i(0), i(n), torch.tensor([n], device="cuda"), src[at].contiguous(), i(0), i(0), to, dst, new, i(1),
                                                       0, n, layer == 0 and k == 0)
                else:
                    lsa.kv_scatter(src[at].contiguous(), to, dst)
        if how == "scatter":
            new[1, :n] = to
        same(pool.view(torch.float8_e4m3fn), scales, new)


@pytest.mark.gpu
def test_rows_at_the_ends_of_bfloat16(lsa):
    """Subnormal rows, the largest finite ones, and both in one row: bits and exponents as defined; read back as the value, to bfloat16's last bit."""
    D = 128
    g = torch.Generator().manual_seed(3)
    x = torch.randn(12, 2, D, generator=g, dtype=torch.float64)
    x = (x / x.abs().amax(-1, keepdim=True)).clamp(-1, 1)
    for t, top in enumerate([2.0 ** -133, 2.0 ** -130, 2.0 ** -127, 2.0 ** -126, 2.0 ** -118, 448 * 2.0 ** -126, 449 * 2.0 ** -126, 2.0 ** -100, 2.0 ** 100, 2.0 ** 127,
                             3.38e38, 3.3895313892515355e38]):
        x[t] *= top
    src = x.to(torch.bfloat16)
    src[-1, 0, 0], src[-1, 1, 1], src[-2, 0, :4] = 3.3895313892515355e38, -3.3895313892515355e38, torch.tensor([2.0 ** -133, -2.0 ** -130, 1.0, 0.0]).to(torch.bfloat16)
    pool = torch.zeros(12, 2, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    sc = torch.zeros(12, 2, dtype=torch.uint8, device="cuda")
    lsa.kv_scatter_fp8(src.cuda(), torch.arange(12, device="cuda"), pool, sc)
    q, e = orc.quantise(src)
    assert torch.equal(pool.cpu().double(), q) and torch.equal(sc.cpu().long(), e)
    assert int(e.min()) == 1 and int(e.max()) == 247
    out = torch.zeros(12, 2, D, dtype=torch.bfloat16, device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lsa.kv_gather_fp8(pool, sc, torch.arange(12, dtype=torch.int32, device="cuda").view(1, 12), i(0), i(12), i(0), 12, out)
    value = q * torch.pow(2.0, (e - 127).double())[..., None]
    want = value.clamp(-3.3895313892515355e38, 3.3895313892515355e38).to(torch.bfloat16).double()
    assert (value.abs() > 3.39e38).any()  # (the largest ones round up to 2^128 as they are written, and come back as the largest bfloat16)
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -133 * (value.abs() < 2.0 ** -126)).all()  # (a step of the subnormal ones)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "e4m3-bf16"])
def test_two_calls_at_once(lsa, kind):
    """Two streams, each with launches of its own that cut the contexts (scratch of their own from the allocator)."""
    cases = [Case(kind, 2, 8, 2, 128, lens, seed=s) for s, lens in ((40, [9000, 77]), (41, [5000, 8000]))]
    want = [[t.clone() for t in c.run(lsa)] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for c, st, g in zip(cases, streams, got):
            with torch.cuda.stream(st):
                g.append(c.run(lsa))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for r in g:
            assert torch.equal(r[0], w[0]) and torch.equal(r[1], w[1])
