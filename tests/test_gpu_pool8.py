"""The KV pool in 8 bits (written, read back, attended over) and decode attention behind a sliding window, against float64."""
import math

import pytest
import torch

from oracle import pool8_oracle as orc

PAD = 2147483647
F8 = torch.float8_e4m3fn


def _rows(shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    return (x * torch.exp(1.5 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)


def _bytes(t):
    return t.view(torch.uint8)


# ------------------------------------------------------------------------------------------------ CPU: the oracle, refusals
def test_oracle_rounds_as_the_format_says():
    """Every e4m3 value stands for itself, halves between neighbours go to the even byte, and torch's conversion agrees."""
    v = orc.e4m3_values()
    assert v[126] == 448 and v[8] == 2.0 ** -6 and v[1] == 2.0 ** -9
    assert torch.equal(orc.round_e4m3(v), v) and torch.equal(orc.round_e4m3(-v), -v)
    mid = (v[1:] + v[:-1]) / 2
    even = torch.where(torch.arange(126) % 2 == 0, v[:-1], v[1:])
    assert torch.equal(orc.round_e4m3(mid), even)
    x = torch.linspace(-448, 448, 4001)
    assert torch.equal(orc.round_e4m3(x.double()).float(), x.to(F8).float())
    q, e = orc.quantise(torch.tensor([[448.0, 1.0], [449.0, 1.0], [0.0, 0.0], [math.inf, 2.0]]))
    assert e.tolist() == [127, 128, 1, 127 - 7] and q[0].tolist() == [448.0, 1.0] and math.isnan(q[3, 0]) and q[3, 1] == 256.0


def test_oracle_window():
    assert orc.visible_positions(10, 3, 2).tolist() == [0, 1, 7, 8, 9]
    assert orc.visible_positions(4, 3, 2).tolist() == [0, 1, 2, 3] and orc.visible_positions(4, None, 0).tolist() == [0, 1, 2, 3]
    assert orc.visible_positions(0, 3, 2).tolist() == [] and orc.visible_positions(5, 1, 0).tolist() == [4]


def test_blocks_match_the_header(tmp_path):
    import ctypes as C
    import os
    import subprocess
    from loongserve_amd import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    blocks = [("lsattn_kv_scatter_fp8_args", _lib.KvScatterFp8Args), ("lsattn_kv_gather_fp8_args", _lib.KvGatherFp8Args),
              ("lsattn_pool_attention_args", _lib.PoolAttentionArgs)]
    lines = []
    for name, cls in blocks:
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f[0]) for f in cls._fields_]
    src = tmp_path / "t.c"
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"lsattn.h\"\nint main(void) {%s return 0;}" % "".join(lines))
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "t")])
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "t")]).split()]
    want = []
    for _, cls in blocks:
        want.append(C.sizeof(cls))
        want += [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want


def test_library_refuses_what_it_cannot_run():
    """Argument checks of the entry points, which launch nothing (the pointers are never followed)."""
    import ctypes as C
    from loongserve_amd import _lib
    lib = _lib.load()

    def write(**kw):
        a = _lib.KvScatterFp8Args(src=4096, src_stride_t=256, src_stride_h=128, dest_index=4096, dest_index_is_i64=1, dtype=0, pool=4096,
                                  pool_stride_0=256, pool_stride_1=128, scales=4096, scale_stride_0=2, scale_stride_1=1, num_tokens=0, num_heads=2,
                                  head_dim=128, num_slots=4)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_kv_scatter_fp8(C.byref(a), None)
    assert write() == 0
    assert write(head_dim=96) == write(dtype=2) == -2
    for bad in (dict(src=None), dict(pool=None), dict(scales=None), dict(dest_index=None), dict(num_tokens=-1), dict(num_heads=0),
                dict(src_stride_t=260), dict(pool_stride_1=120), dict(pool=4097), dict(dest_index_is_i64=2)):
        assert write(**bad) == -1, bad

    def read(**kw):
        a = _lib.KvGatherFp8Args(pool=4096, pool_stride_0=256, pool_stride_1=128, scales=4096, scale_stride_0=2, scale_stride_1=1, num_slots=4,
                                 req_to_tokens=4096, num_reqs=2, max_seq_len=8, b_req_idx=4096, b_seq_len=4096, b_start_loc=4096, batch=0,
                                 max_len_in_batch=8, out=4096, out_stride_t=256, out_stride_h=128, out_rows=8, dtype=0, num_heads=2, head_dim=128)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_kv_gather_fp8(C.byref(a), None)
    assert read() == 0 and read(batch=3, max_len_in_batch=0) == 0
    assert read(head_dim=48) == read(dtype=2) == -2
    for bad in (dict(pool=None), dict(out=None), dict(b_start_loc=None), dict(batch=-1), dict(batch=65536), dict(out_stride_t=4), dict(out=4104 + 1),
                dict(num_slots=-1), dict(max_len_in_batch=-1)):
        assert read(**bad) == -1, bad

    def attend(**kw):
        a = _lib.PoolAttentionArgs(q=4096, k=4096, v=4096, k_stride_0=256, k_stride_1=128, v_stride_0=256, v_stride_1=128, k_scales=4096, v_scales=4096,
                                   ks_stride_0=2, ks_stride_1=1, vs_stride_0=2, vs_stride_1=1, req_to_tokens=4096, b_req_idx=4096, b_seqlen=4096,
                                   batch=0, num_q_heads=4, num_kv_heads=2, head_dim=128, num_slots=4, num_reqs=2, max_seq_len=8, max_len_in_batch=8,
                                   window=0, sinks=0, dtype=0, kv_dtype=3, sm_scale=0.1, o_dtype=2, o=4096, lse=4096)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_pool_attention(C.byref(a), None)
    assert attend() == 0 and attend(kv_dtype=0) == 0 and attend(dtype=1, kv_dtype=1) == 0
    assert attend(head_dim=96) == attend(num_q_heads=5) == attend(dtype=0, kv_dtype=1) == attend(dtype=2) == attend(o_dtype=3) == -2
    for bad in (dict(q=None), dict(lse=None), dict(k_scales=None), dict(window=-1), dict(sinks=-1), dict(batch=-1), dict(k_stride_0=250),
                dict(num_slots=0), dict(sm_scale=0.0), dict(v=4100), dict(batch=65536)):
        assert attend(**bad) == -1, bad
    assert attend(batch=2, max_len_in_batch=1 << 20) == -4  # (partials, and no workspace)
    size = lib.lsattn_pool_attention_workspace_bytes
    assert size(2, 4, 2, 128, 1 << 20, 0, 0) > 0 and size(2, 4, 2, 128, 1 << 20, 512, 4) == 0 and size(0, 4, 2, 128, 9, 0, 0) == 0
    assert size(2, 4, 2, 128, 1 << 20, 2 ** 63 - 1, 9) == size(2, 4, 2, 128, 1 << 20, 9, 2 ** 63 - 1) == size(2, 4, 2, 128, 1 << 20, 0, 0)


def test_python_operators_refuse_cpu_tensors():
    import loongserve_amd as lsa
    x, i = torch.zeros(2, 4, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    pool, sc, table = torch.zeros(8, 4, 128).to(F8), torch.zeros(8, 4, dtype=torch.uint8), torch.zeros(2, 8, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        lsa.kv_scatter_fp8(x, i, pool, sc)
    with pytest.raises(ValueError, match="GPU"):
        lsa.kv_gather_fp8(pool, sc, table, i, i, i, 1, x)
    with pytest.raises(ValueError, match="GPU"):
        lsa.longserve_fp8_decode_attention(x, table, i, i, 8, pool[:, :2], pool[:, 2:], sc[:, :2], sc[:, 2:])
    with pytest.raises(ValueError, match="GPU"):
        lsa.longserve_window_decode_attention(x, table, i, i, 8, x[:, :2], x[:, 2:], 4)
    with pytest.raises(ValueError, match="window"):
        lsa.longserve_window_decode_attention(x, table, i, i, 8, x[:, :2], x[:, 2:], None)


# ------------------------------------------------------------------------------------------------ writing
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,D,i64", [(1, 2, 128, True), (7, 16, 128, False), (33, 6, 64, True), (5, 3, 32, False), (9, 10, 16, True), (257, 64, 128, True)])
def test_write_is_the_definition_bit_for_bit(lsa, dtype, T, H, D, i64):
    x = _rows((T, H, D), T * 31 + D, dtype)
    x[0, 0] = 0
    x[-1, -1, :3] = torch.tensor([448.0, 449.0, -1.0]).to(dtype)
    x[T // 2, H // 2] *= 1e-4  # (subnormal in fp16)
    slots = T + 5
    idx = torch.randperm(slots, generator=torch.Generator().manual_seed(1))[:T]
    pool = torch.full((slots, H, D), 3.0).to(F8).cuda()
    sc = torch.full((slots, H), 77, dtype=torch.uint8, device="cuda")
    lsa.kv_scatter_fp8(x.cuda(), (idx if i64 else idx.int()).cuda(), pool, sc)
    q, e = orc.quantise(x)
    want, want_sc = torch.full((slots, H, D), 3.0), torch.full((slots, H), 77)
    want[idx], want_sc[idx] = q.float(), e
    assert torch.equal(pool.cpu().float(), want) and torch.equal(sc.cpu().long(), want_sc)


@pytest.mark.gpu
def test_write_of_what_is_not_finite_strided_rows_and_slots_outside(lsa):
    T, H, D = 6, 4, 128
    big = _rows((T, 2 * H, D + 8), 3, torch.float16).cuda()
    src = big[:, 2:2 + H, 8:8 + D]  # a strided view, 16-byte aligned
    src[1, 0, 5], src[1, 0, 6], src[2, 3, 0] = math.nan, math.inf, -math.inf
    src[3, 2] = math.nan
    store = torch.zeros(9, 3 * H, 2 * D, device="cuda").to(F8)
    pool, sc_store = store[:, H:2 * H, :D], torch.zeros(9, 5 * H, dtype=torch.uint8, device="cuda")
    sc = sc_store[:, 1:1 + 2 * H:2]
    idx = torch.tensor([8, 0, PAD, 3, -1, 5], dtype=torch.int32, device="cuda")
    lsa.kv_scatter_fp8(src, idx, pool, sc)
    q, e = orc.quantise(src.cpu())
    want, want_sc = torch.zeros(9, H, D), torch.zeros(9, H, dtype=torch.int64)
    for t, s in enumerate(idx.tolist()):
        if 0 <= s < 9:
            want[s], want_sc[s] = q[t].float(), e[t]
    assert torch.equal(pool.cpu().float().nan_to_num(1e9), want.nan_to_num(1e9)) and torch.equal(sc.cpu().long(), want_sc)
    assert not _bytes(store[:, :H]).any() and not _bytes(store[:, :, D:]).any() and not sc_store[:, 0::2].any()  # nothing beside them


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,D,lens", [(16, 128, [5, 0, 1, 300]), (2, 64, [64, 33]), (3, 32, [7]), (64, 128, [20, 21]), (1, 16, [1000])])
def test_read_back_and_rows_left_alone(lsa, dtype, H, D, lens):
    n = sum(lens)
    x = _rows((n + 8, H, D), 5 + D, dtype)
    q, e = orc.quantise(x)
    perm = torch.randperm(n + 8, generator=torch.Generator().manual_seed(2))
    pool, sc = q.float().to(F8).cuda()[perm.argsort()], e.to(torch.uint8).cuda()[perm.argsort()]
    value = (q * torch.pow(2.0, (e - 127).double())[..., None])[perm.argsort()]
    first = [i % 3 for i in range(len(lens))]
    table = torch.full((len(lens) + 2, max(lens) + 3), PAD, dtype=torch.int32)
    req = torch.arange(len(lens) + 2, dtype=torch.int32).flip(0)[:len(lens)].contiguous()
    at, slots = 0, []
    for b, m in enumerate(lens):
        s = torch.arange(at, at + m, dtype=torch.int32)
        table[req[b], first[b]:first[b] + m] = s
        slots.append(s)
        at += m
    if lens[-1] > 4:
        table[req[-1], first[-1] + 2] = PAD  # a hole: a row of zeros
    start = torch.tensor([2 + sum(lens[:b]) for b in range(len(lens))], dtype=torch.int32)
    out = torch.full((n + 6, H, D), 9.0, dtype=dtype, device="cuda")
    lsa.kv_gather_fp8(pool, sc, table.cuda(), req.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), start.cuda(), max(lens), out,
                      torch.tensor(first, dtype=torch.int32, device="cuda"))
    want = torch.full((n + 6, H, D), 9.0, dtype=torch.float64)
    for b, m in enumerate(lens):
        want[start[b]:start[b] + m] = value[slots[b].long()]
    if lens[-1] > 4:
        want[start[-1] + 2] = 0
    assert torch.equal(out.cpu().double(), want.to(dtype).double())


@pytest.mark.gpu
def test_read_back_of_values_past_fp16_and_outside_the_buffers(lsa):
    x = torch.full((2, 1, 128), 65504.0, dtype=torch.float16)
    x[0, 0, 1], x[1, 0, 0] = -65504.0, math.nan
    pool, sc = torch.zeros(2, 1, 128, device="cuda").to(F8), torch.zeros(2, 1, dtype=torch.uint8, device="cuda")
    lsa.kv_scatter_fp8(x.cuda(), torch.arange(2, device="cuda"), pool, sc)
    out = torch.full((4, 1, 128), 5.0, dtype=torch.float16, device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    table = i(0, 1, 0, 1).view(1, 4)
    # four tokens, of which the first lies in front of out; a request that the table has not
    lsa.kv_gather_fp8(pool, sc, table, i(0, 7), i(4, 1), i(-1, 3), 4, out)
    o = out.cpu()
    assert math.isnan(o[0, 0, 0]) and (o[0, 0, 1:] == 65504).all()
    assert o[1, 0, 0] == 65504 and o[1, 0, 1] == -65504 and torch.equal(o[2].nan_to_num(1), o[0].nan_to_num(1)) and not o[3].any()
    big = torch.full((4, 1, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    lsa.kv_gather_fp8(pool, sc, table, i(0), i(9), i(1), 9, big)  # (past the table's width: zeros; past out: not written)
    assert (big[0] == 5).all() and big[1, 0, 0] == 65536 and big[3, 0, 0] == 65536


@pytest.mark.gpu
def test_read_back_stops_at_the_longest_length_given(lsa):
    """A request longer than the bound: the rows behind it stay as they were, also those that the last workgroup could reach."""
    for H, D in ((1, 16), (3, 64), (40, 128)):
        pool, sc = torch.zeros(40, H, D, device="cuda").to(F8), torch.full((40, H), 127, dtype=torch.uint8, device="cuda")
        out = torch.full((40, H, D), 5.0, dtype=torch.float16, device="cuda")
        i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        lsa.kv_gather_fp8(pool, sc, torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40), i(0, 0), i(30, 2), i(0, 20), 7, out)
        want = torch.full((40, H, D), 5.0, dtype=torch.float16)
        want[:7] = want[20:22] = 0
        assert torch.equal(out.cpu(), want)


# ------------------------------------------------------------------------------------------------ decode
KINDS = {"f16": (torch.float16, None), "bf16": (torch.bfloat16, None), "e4m3-f16": (torch.float16, F8), "e4m3-bf16": (torch.bfloat16, F8)}


class Case:
    def __init__(self, kind, B, Hq, Hkv, D, lens, seed=0, extra=40, holes=()):
        dtype, kv = KINDS[kind]
        g = torch.Generator().manual_seed(seed * 1000 + Hq + D)
        n = sum(max(m, 0) for m in lens) + extra
        self.dtype, self.k8, self.Hkv, self.lens, self.D = dtype, kv is not None, Hkv, lens, D
        self.q = torch.randn(B, Hq, D, generator=g).to(dtype)
        rows = _rows((n, 2 * Hkv, D), seed + 7, dtype)
        rows[:, :Hkv] = torch.randn(n, Hkv, D, generator=g).to(dtype)
        width = max(max(lens), 1) + 3
        self.table = torch.full((B + 2, width), PAD, dtype=torch.int32)
        self.req = torch.randperm(B + 2, generator=g)[:B].to(torch.int32)
        perm = torch.randperm(n, generator=g).to(torch.int32)
        at = 0
        for b, m in enumerate(lens):
            if m > 0:
                self.table[self.req[b], :m] = perm[at:at + m]
                at += m
        for b, pos in holes:
            self.table[self.req[b], pos] = (PAD, -1, n)[pos % 3]
        unused = perm[at:]
        if self.k8:
            q, e = orc.quantise(rows)
            self.values = q * torch.pow(2.0, (e - 127).double())[..., None]
            self.pool = q.float().to(F8)
            self.pool.view(torch.uint8)[unused.long()] = 0x7F  # NaN where no request looks
            self.scales = e.to(torch.uint8).cuda()
        else:
            self.values, self.pool, self.scales = rows.double(), rows.clone(), None
            self.pool[unused.long()] = math.nan
        self.pool = self.pool.cuda()
        self.len = torch.tensor(lens, dtype=torch.int32)

    def run(self, lsa, window=None, sinks=0, max_len=None, **kw):
        h = self.Hkv
        a = (self.q.cuda(), self.table.cuda(), self.req.cuda(), self.len.cuda(), max(self.lens) if max_len is None else max_len, self.pool[:, :h], self.pool[:, h:])
        if self.k8:
            return lsa.longserve_fp8_decode_attention(*a, self.scales[:, :h], self.scales[:, h:], window=window, sinks=sinks, **kw)
        return lsa.longserve_window_decode_attention(*a, 1 << 30 if window is None else window, sinks, **kw)

    def check(self, got, window=None, sinks=0, half=0.0):
        h = self.Hkv
        o, lse, tol_o, tol_l = orc.decode(self.q, self.values[:, :h], self.values[:, h:], self.table, self.req, self.len, window, sinks)
        g, l = got[0].cpu().double(), got[1].cpu().double()
        assert torch.isfinite(g).all()
        assert ((g - o).abs() <= tol_o + half * (o.abs() + tol_o) + (1e-30 if not half else 2.0 ** -24)).all(), (g - o).abs().max()
        fin = torch.isfinite(lse)
        assert torch.equal(fin, torch.isfinite(l)) and ((l - lse).abs() <= tol_l)[fin].all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (5, 1, 128), (24, 2, 128), (9, 1, 64), (32, 8, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (64, 4), (33, 100)])
def test_decode_short(lsa, kind, Hq, Hkv, D, window, sinks):
    c = Case(kind, 6, Hq, Hkv, D, [1, 0, 33, 97, 32, 700], seed=Hq)
    c.check(c.run(lsa, window, sinks), window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("Hq,Hkv,lens,window,sinks", [(4, 1, [12000], None, 0), (8, 2, [9000, 0, 1, 40, 5000, 64], None, 0), (12, 1, [4097, 3], 5000, 3),
                                                      (2, 2, [9500, 31], 4090, 77)])
def test_decode_long_and_ragged(lsa, kind, Hq, Hkv, lens, window, sinks):
    c = Case(kind, len(lens), Hq, Hkv, 128, lens, seed=len(lens))
    c.check(c.run(lsa, window, sinks), window, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "e4m3-bf16"])
def test_decode_with_more_requests_than_lanes(lsa, kind):
    """A batch of more than 64 requests, long enough to be cut: a wave counts the requests in steps of 64."""
    lens = [(i * 37) % 90 for i in range(150)]
    lens[70] = 9000
    c = Case(kind, 150, 4, 2, 64, lens, seed=3)
    c.check(c.run(lsa))
    c.check(c.run(lsa, max_len=1 << 17))  # (the bound only steers)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "e4m3-f16"])
@pytest.mark.parametrize("lens,holes", [([70, 40], [(0, 0), (0, 33), (0, 34), (1, 39)]), ([9000, 3], [(0, 0), (0, 8999), (0, 4000), (0, 4001), (1, 0), (1, 1), (1, 2)])])
def test_entries_outside_the_pool_do_not_exist(lsa, kind, lens, holes):
    c = Case(kind, 2, 8, 2, 128, lens, seed=5, holes=holes)
    c.check(c.run(lsa))
    c.check(c.run(lsa, 50, 3), 50, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "e4m3-f16", "e4m3-bf16"])
@pytest.mark.parametrize("lens", [[200, 31], [9000]])
def test_decode_outputs_in_16_bits_given_buffers_and_workspace(lsa, kind, lens):
    c = Case(kind, len(lens), 8, 2, 128, lens, seed=6)
    for dt, half in ((torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8), (torch.float32, 0.0)):
        out, lse = torch.empty(c.q.shape, dtype=dt, device="cuda"), torch.empty(c.q.shape[:2], device="cuda")
        need = lsa.pool_attention_workspace_bytes(len(lens), 8, 2, 128, max(lens), None if c.k8 else 1 << 30)
        ws = torch.full((need // 4 + 4,), math.nan, device="cuda")
        got = c.run(lsa, out=out, o_logexpsum=lse, workspace=ws)
        assert got[0] is out and got[1] is lse
        c.check(got, half=half)
    if need:
        with pytest.raises(ValueError, match="workspace"):
            c.run(lsa, workspace=ws[:need // 4 - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[70, 31], [9000]])
def test_windows_as_wide_as_integers_go(lsa, lens):
    c = Case("f16", len(lens), 4, 2, 128, lens, seed=8)
    for window, sinks in ((2 ** 63 - 1, 5), (2 ** 63 - 1, 2 ** 63 - 1), (9, 2 ** 63 - 1), (2 ** 31 - 1, 2 ** 31 - 1)):
        c.check(c.run(lsa, window, sinks))


@pytest.mark.gpu
def test_decode_refusals_on_the_gpu(lsa):
    c = Case("e4m3-f16", 2, 8, 2, 128, [20, 9])
    for kw in (dict(window=0), dict(window=-3), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError, match="window"):
            c.run(lsa, **kw)
    with pytest.raises(ValueError, match="out must"):
        c.run(lsa, out=torch.empty(2, 8, 64, device="cuda"))
    q, i = c.q.cuda(), c.len.cuda()
    with pytest.raises(ValueError, match="type of q"):
        lsa.longserve_window_decode_attention(q, c.table.cuda(), i, i, 20, c.pool[:, :2], c.pool[:, 2:], 4)
    with pytest.raises(ValueError, match="float8"):
        lsa.longserve_fp8_decode_attention(q, c.table.cuda(), i, i, 20, c.pool[:, :2].half(), c.pool[:, 2:].half(), c.scales[:, :2], c.scales[:, 2:])
    with pytest.raises(ValueError, match="b_req_idx"):
        lsa.longserve_fp8_decode_attention(q, c.table.cuda(), i.long(), i, 20, c.pool[:, :2], c.pool[:, 2:], c.scales[:, :2], c.scales[:, 2:])
    with pytest.raises(ValueError, match="slots and heads"):
        lsa.kv_scatter_fp8(q, i, c.pool[:, :2], c.scales)
    with pytest.raises(ValueError, match="rows must match"):
        lsa.kv_scatter_fp8(q, i, c.pool, c.scales)
    with pytest.raises(ValueError, match="dest_index"):
        lsa.kv_scatter_fp8(q[:, :4], i[:1], c.pool, c.scales)
    with pytest.raises(ValueError, match="out must"):
        lsa.kv_gather_fp8(c.pool, c.scales, c.table.cuda(), i, i, i, 4, q)


@pytest.mark.gpu
def test_scores_and_scales_at_the_ends_of_their_range(lsa):
    """K and V of very different sizes from token to token, and scores in the hundreds: one token takes all the weight, or the V of a token with
    little weight counts as much as the others'."""
    for kind in ("e4m3-f16", "e4m3-bf16", "f16", "bf16"):
        c = Case(kind, 2, 8, 2, 128, [300, 90], seed=8)
        big = 2.0 ** 10 if kind != "f16" else 2.0 ** 6
        factor = torch.where(torch.arange(c.values.shape[0]) % 7 == 0, big, 2.0 ** -8 if c.k8 else 1.0).double()
        c.values = c.values.clone()
        if c.k8:
            c.values *= factor[:, None, None]
            c.scales += torch.log2(factor).to(torch.int8).cuda()[:, None].to(torch.uint8)
        else:
            c.values[:, 2:] *= factor[:, None, None]
            c.pool = torch.where(torch.isnan(c.pool), c.pool, c.values.to(c.dtype).cuda())
            c.values = c.values.to(c.dtype).double()
        c.check(c.run(lsa))


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[300, 31], [9000, 20]])
def test_decode_on_a_stream_of_its_own_and_captured(lsa, lens):
    """The call on another stream, and recorded into a graph that is replayed on new inputs between eager calls."""
    c = Case("e4m3-f16", 2, 8, 2, 128, lens, seed=9)
    h = 2
    q, table, req, n = c.q.cuda(), c.table.cuda(), c.req.cuda(), c.len.cuda()
    call = lambda: lsa.longserve_fp8_decode_attention(q, table, req, n, max(lens), c.pool[:, :h], c.pool[:, h:], c.scales[:, :h], c.scales[:, h:])  # noqa: E731
    eager = [t.clone() for t in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for seed in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).half())
        n.copy_(torch.tensor([max(1, lens[0] - 50 * seed), lens[1] - seed], dtype=torch.int32))
        eager = [t.clone() for t in call()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, eager)), seed


@pytest.mark.gpu
def test_a_layer_over_the_8_bit_pool(lsa):
    """Slots from the allocator, a prompt written and registered, the next chunk behind its context read back, decode steps behind a window and
    without, and the rows moved to other slots with their exponents: every output against float64 over the values that the pool stands for."""
    Hq, Hkv, D, L0, L1 = 8, 2, 128, 150, 41
    mem = lsa.LongServeMemoryManager(600, F8, Hkv, D, 1)
    req = lsa.LongServeReqManager(4, 400, mem)
    pool, sc = mem.kv_buffer[0], mem.kv_scales[0]
    assert pool.dtype == F8 and sc.shape == (600, 2 * Hkv)
    r = req.alloc(1).int()
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    rows = _rows((L0 + L1 + 3, 2 * Hkv, D), 11, torch.float16).cuda()
    mem.alloc(37)  # (so that the slots are not 0, 1, ...)
    slots = mem.alloc(L0)
    lsa.kv_scatter_fp8(rows[:L0], slots, pool, sc)
    lsa.init_req_to_token_indexes(req.req_to_token_indexs, r, i(L0), slots, i(0), L0)
    kept, e = orc.quantise(rows.cpu())
    kept = kept * torch.pow(2.0, (e - 127).double())[..., None]
    # the next chunk: the context back, the chunk's own rows behind it
    kv = torch.empty(L0 + L1, 2 * Hkv, D, dtype=torch.float16, device="cuda")
    lsa.kv_gather_fp8(pool, sc, req.req_to_token_indexs, r, i(L0), i(0), L0, kv)
    assert torch.equal(kv[:L0].cpu().double(), kept[:L0])
    kv[L0:] = rows[L0:L0 + L1]
    q = torch.randn(L1, Hq, D, device="cuda").half()
    o, lse = lsa.prefill_attention_step(q, kv[:, :Hkv], kv[:, Hkv:], i(0), i(L1), i(L0), i(0), i(L0 + L1), i(0), 1, L1)
    s = torch.einsum("mhd,nhd->hmn", q.cpu().double(), kv[:, :Hkv].cpu().double().repeat_interleave(4, 1)) / math.sqrt(D)
    s = s.masked_fill(torch.arange(L0 + L1)[None] > L0 + torch.arange(L1)[:, None], -math.inf)
    want = torch.einsum("hmn,nhd->mhd", torch.softmax(s, -1), kv[:, Hkv:].cpu().double().repeat_interleave(4, 1))
    assert ((o.cpu().double() - want).norm() / want.norm()) < 1e-3
    slots = mem.alloc(L1)
    lsa.kv_scatter_fp8(rows[L0:L0 + L1], slots, pool, sc)
    req.req_to_token_indexs[r.long(), L0:L0 + L1] = slots.int()
    for step in range(3):
        n = L0 + L1 + step + 1
        slot = mem.alloc(1)
        lsa.kv_scatter_fp8(rows[n - 1:n], slot, pool, sc)
        lsa.copy_kv_index_to_req(req.req_to_token_indexs, r, i(n), slot)
        qd = torch.randn(1, Hq, D, device="cuda").half()
        for window, sinks in ((None, 0), (64, 4)):
            got = lsa.longserve_fp8_decode_attention(qd, req.req_to_token_indexs, r, i(n), n, pool[:, :Hkv], pool[:, Hkv:], sc[:, :Hkv], sc[:, Hkv:],
                                                     window=window, sinks=sinks)
            o, lse, tol_o, tol_l = orc.decode(qd.cpu(), kept[:n, :Hkv], kept[:n, Hkv:], torch.arange(n)[None], [0], [n], window, sinks)
            assert ((got[0].cpu().double() - o).abs() <= tol_o).all() and ((got[1].cpu().double() - lse).abs() <= tol_l).all()
    # the same rows in other slots: moved with their exponents, the same result bit for bit
    new = mem.alloc(n)
    old = req.req_to_token_indexs[r.long(), :n].long().flatten()
    lsa.kv_scatter(_bytes(pool)[old], new, _bytes(pool))
    sc[new] = sc[old]
    req.req_to_token_indexs[r.long(), :n] = new.int()
    again = lsa.longserve_fp8_decode_attention(qd, req.req_to_token_indexs, r, i(n), n, pool[:, :Hkv], pool[:, Hkv:], sc[:, :Hkv], sc[:, Hkv:], window=64, sinks=4)
    assert all(torch.equal(x, y) for x, y in zip(again, got))
    assert mem.kv_scales is not None and lsa.LongServeMemoryManager(8, torch.float16, 1, 16, 1).kv_scales is None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("lens", [[0, 0, 0], [0, 0, 1]])
def test_batches_without_tokens(lsa, kind, lens):
    """Padded batches, in both launch forms (the bound only steers)."""
    c = Case(kind, 3, 8, 2, 128, lens, seed=9)
    for max_len in (0, 64, 1 << 17):
        got = c.run(lsa, max_len=max_len)
        c.check(got)
        assert not got[0][:2].any() and (got[1][:2] == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [300, 9000])
def test_slots_past_four_gigabytes(lsa, n):
    """A pool whose last slots lie more than 2^32 bytes (8 bits) and 2^33 bytes (16 bits) behind its first."""
    Hkv, D, slots = 8, 128, (1 << 21) + 12000  # 2 KB a slot in 8 bits
    x = _rows((n, 2 * Hkv, D), 3, torch.float16)
    where = (slots - 1 - torch.randperm(n, generator=torch.Generator().manual_seed(1))).to(torch.int32)
    table = where.view(1, n).cuda()
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = _rows((1, 16, D), 4, torch.float16)
    pool, sc = torch.empty(slots, 2 * Hkv, D, dtype=F8, device="cuda"), torch.empty(slots, 2 * Hkv, dtype=torch.uint8, device="cuda")
    lsa.kv_scatter_fp8(x.cuda(), where.cuda(), pool, sc)
    want, e = orc.quantise(x)
    value = want * torch.pow(2.0, (e - 127).double())[..., None]
    out = torch.empty(n, 2 * Hkv, D, dtype=torch.float16, device="cuda")
    lsa.kv_gather_fp8(pool, sc, table, i(0), i(n), i(0), n, out)
    assert torch.equal(out.cpu().double(), value.to(torch.float16).double())
    near = torch.zeros(1, n, dtype=torch.int32)
    near[0] = torch.arange(n)
    for k8 in (True, False):
        if k8:
            got = lsa.longserve_fp8_decode_attention(q.cuda(), table, i(0), i(n), n, pool[:, :Hkv], pool[:, Hkv:], sc[:, :Hkv], sc[:, Hkv:])
        else:
            del pool
            pool = torch.empty(slots, 2 * Hkv, D, dtype=torch.float16, device="cuda")
            lsa.kv_scatter(x.cuda(), where.cuda(), pool)
            got = lsa.longserve_window_decode_attention(q.cuda(), table, i(0), i(n), n, pool[:, :Hkv], pool[:, Hkv:], n, 0)
        rows = value if k8 else x.double()
        o, lse, tol_o, tol_l = orc.decode(q, rows[:, :Hkv], rows[:, Hkv:], near, torch.zeros(1, dtype=torch.int32), torch.tensor([n], dtype=torch.int32), None, 0)
        assert ((got[0].cpu().double() - o).abs() <= tol_o + 1e-30).all() and ((got[1].cpu().double() - lse).abs() <= tol_l).all()
