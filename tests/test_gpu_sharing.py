"""Requests that share tokens of the pool: attention over shared prefixes, forks, releases and compaction, against float64 and plain restatements."""
import math

import pytest
import torch

from oracle import sharing_oracle as orc

PAD = 2147483647
F8 = torch.float8_e4m3fn
DEV = "cuda:0"


# ------------------------------------------------------------------------------------------------ CPU: blocks, refusals, the oracle
def test_blocks_match_the_header(tmp_path):
    import ctypes as C
    import os
    import subprocess
    from loongserve_amd import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    blocks = [("lsattn_shared_decode_args", _lib.SharedDecodeArgs), ("lsattn_shared_prefill_args", _lib.SharedPrefillArgs), ("lsattn_pool_rows", _lib.PoolRows),
              ("lsattn_copy_requests_args", _lib.CopyRequestsArgs), ("lsattn_compact_args", _lib.CompactArgs)]
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
    P = 4096

    def decode(**kw):
        a = _lib.SharedDecodeArgs(q=P, k=P, v=P, k_stride_0=256, k_stride_1=128, v_stride_0=256, v_stride_1=128, req_to_tokens=P, b_req_idx=P, b_seqlen=P,
                                  g_start_loc=P, g_size=P, g_req_idx=P, g_prefix_len=P, batch=0, num_groups=1, num_q_heads=4, num_kv_heads=2, head_dim=128,
                                  num_slots=4, num_reqs=2, max_seq_len=8, max_prefix_len=4, max_own_len=4, dtype=0, o_dtype=0, sm_scale=0.1, o=P, lse=P)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_shared_decode(C.byref(a), None)
    assert decode() == 0 and decode(dtype=1, o_dtype=2) == 0 and decode(num_groups=0, g_start_loc=None) == 0
    assert decode(head_dim=96) == decode(num_q_heads=5) == decode(dtype=2) == decode(o_dtype=3) == -2
    for bad in (dict(q=None), dict(lse=None), dict(o=None), dict(g_size=None), dict(batch=-1), dict(num_groups=-1), dict(max_prefix_len=-1), dict(max_own_len=-1),
                dict(k_stride_0=250), dict(num_slots=0), dict(sm_scale=0.0), dict(sm_scale=math.nan), dict(v=P + 4), dict(batch=65536), dict(k_stride_0=-256)):
        assert decode(**bad) == -1, bad
    assert decode(batch=3) == -4  # no workspace
    need = lib.lsattn_shared_decode_workspace_bytes(3, 1, 4, 2, 128, 4, 4)
    assert need > 0 and decode(batch=3, workspace=P, workspace_bytes=need - 1) == -4 and decode(batch=3, workspace=P + 4, workspace_bytes=need) == -1
    for bad in ((0, 1, 4, 2, 128, 4, 4), (3, -1, 4, 2, 128, 4, 4), (3, 1, 4, 3, 128, 4, 4), (3, 1, 4, 2, 80, 4, 4), (3, 1, 4, 2, 128, -1, 4), (70000, 1, 4, 2, 128, 4, 4)):
        assert lib.lsattn_shared_decode_workspace_bytes(*bad) == 0, bad

    def prompt(**kw):
        a = _lib.SharedPrefillArgs(q=P, q_stride_t=512, q_stride_h=128, k=P, v=P, k_stride_0=256, k_stride_1=128, v_stride_0=256, v_stride_1=128, req_to_tokens=P,
                                   g_start_loc=P, g_size=P, g_req_idx=P, g_prefix_len=P, rows=0, num_groups=1, num_q_heads=4, num_kv_heads=2, head_dim=128,
                                   num_slots=4, num_reqs=2, max_seq_len=8, max_prefix_len=4, max_group_rows=4, dtype=0, sm_scale=0.1, o=P, o_stride_t=512,
                                   o_stride_h=128, m=P, l=P, ml_stride_t=4, ml_stride_h=1)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_shared_prefill(C.byref(a), None)
    assert prompt() == 0 and prompt(dtype=1) == 0 and prompt(rows=5, num_groups=0) == 0 and prompt(rows=5, max_prefix_len=0) == 0
    assert prompt(head_dim=32) == prompt(num_q_heads=5) == prompt(dtype=2) == -2
    for bad in (dict(q=None), dict(m=None), dict(o=None), dict(g_req_idx=None), dict(rows=-1), dict(max_group_rows=-1), dict(q_stride_t=516), dict(o_stride_h=4),
                dict(num_slots=0), dict(sm_scale=-1.0), dict(k=P + 8), dict(num_groups=65536), dict(m=P + 2)):
        assert prompt(**bad) == -1, bad
    for rows in (5, 5000):
        need = lib.lsattn_shared_prefill_workspace_bytes(rows, 1, 4, 2, 128, 4)
        assert need > 0 and prompt(rows=rows) == -4 and prompt(rows=rows, workspace=P, workspace_bytes=need - 1) == -4
        assert prompt(rows=rows, workspace=P + 8, workspace_bytes=need) == -1

    assert lib.lsattn_fork_requests(P, 2, 8, P, P, P, 0, 8, P, 4, None) == 0
    for bad in ((None, 2, 8, P, P, P, 0, 8, P, 4), (P, -1, 8, P, P, P, 0, 8, P, 4), (P, 2, 8, P, None, P, 0, 8, P, 4), (P, 2, 8, P, P, P, 65536, 8, P, 4),
                (P, 2, 8, P, P, P, 1, -1, P, 4), (P, 2, 8, P, P, P, 1, 8, None, 4), (P, 2, 8, P, P, P, 1, 8, P, -1)):
        assert lib.lsattn_fork_requests(*bad, None) == -1, bad

    def rows_of(**kw):
        r = _lib.PoolRows(rows=P, layer_stride_bytes=1024, slot_stride_bytes=256, row_bytes=256, num_layers=2, num_slots=4)
        for k, x in kw.items():
            setattr(r, k, x)
        return r

    def copy(r=None, **kw):
        a = _lib.CopyRequestsArgs(req_to_tokens=P, num_reqs=2, max_seq_len=8, src_req_idx=P, dst_req_idx=P, b_seq_len=P, b_start_loc=P, n=0, max_len_in_batch=8,
                                  mem_index=P, num_index=4)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_copy_requests(C.byref(a), C.byref(r or rows_of()), None)
    assert copy() == 0 and copy(rows_of(scales=P, scale_bytes=2, scale_slot_stride_bytes=2, scale_layer_stride_bytes=8)) == 0
    for bad in (dict(rows=None), dict(row_bytes=24), dict(row_bytes=0), dict(slot_stride_bytes=128), dict(num_layers=0), dict(num_slots=0), dict(rows=P + 8),
                dict(scales=P), dict(scales=P, scale_bytes=4, scale_slot_stride_bytes=2)):
        assert copy(rows_of(**bad)) == -1, bad
    for bad in (dict(req_to_tokens=None), dict(mem_index=None), dict(n=-1), dict(n=65536), dict(num_index=-1), dict(max_len_in_batch=-1)):
        assert copy(**bad) == -1, bad

    release = lambda *a: lib.lsattn_release_requests(*a, None)  # noqa: E731
    for bad in ((None, 2, 8, P, P, 1, 8, P, 4, P, None, 0), (P, 2, 8, P, P, -1, 8, P, 4, P, None, 0), (P, 2, 8, P, P, 1, 8, None, 4, P, None, 0),
                (P, 2, 8, P, P, 1, 8, P, 4, None, None, 0), (P, 2, 8, P, P, 65536, 8, P, 4, P, None, 0)):
        assert release(*bad) == -1, bad
    need = lib.lsattn_release_workspace_bytes(100, 5000)
    assert need > 0 and release(P, 200, 6000, P, P, 100, 5000, P, 4, P, P, need - 1) == -4 and release(P, 200, 6000, P, P, 100, 5000, P, 4, P, None, need) == -4

    def compact(r=None, **kw):
        a = _lib.CompactArgs(mem_state=P, pool_size=0, remap=P, req_to_tokens=P, num_reqs=2, max_seq_len=8, b_req_idx=P, b_seq_len=P, n=1, max_len_in_batch=8)
        for k, x in kw.items():
            setattr(a, k, x)
        return lib.lsattn_compact_pool(C.byref(a), C.byref(r or rows_of()), None)
    assert compact() == 0
    for bad in (dict(pool_size=-1), dict(n=-1), dict(pool_size=5), dict(pool_size=4, mem_state=None), dict(pool_size=4, remap=None), dict(pool_size=4, b_req_idx=None)):
        assert compact(**bad) == -1, bad
    assert compact(pool_size=4) == -4 and lib.lsattn_compact_workspace_bytes(0) == 0


def test_operators_refuse_tensors_that_are_not_on_the_gpu():
    import loongserve_amd as lsa
    i = torch.zeros(2, dtype=torch.int32)
    t, q, kv, st = torch.zeros(2, 8, dtype=torch.int32), torch.zeros(2, 4, 128).half(), torch.zeros(8, 2, 128).half(), torch.zeros(8, dtype=torch.int32)
    m = torch.zeros(2, 4)
    for call in (lambda: lsa.longserve_shared_prefix_decode_attention(q, t, i, i, 8, kv, kv, i, i, i, i, 4),
                 lambda: lsa.shared_prefix_attention_fwd(q, kv, kv, q, i, i, t, i, i, 2, 4, m, m),
                 lambda: lsa.fork_requests(t, i, i, i, 8, st),
                 lambda: lsa.copy_requests(t, i, i, i, i, 8, i.long(), kv[None], None),
                 lambda: lsa.release_requests(t, i, i, 8, st),
                 lambda: lsa.compact_pool(st, kv[None], t, i, i, 8)):
        with pytest.raises(ValueError, match="must live on the GPU"):
            call()


def test_oracle_groups_and_compaction():
    assert orc.members([0, 1, 5], [3, 3, 9], [0, 1, 9], [4, 5, 6], 7, 3, 10) == ([0, 0, 0, 1, -1, 2, 2], [4, 4, 4, 5, 0, 0, 0])
    assert orc.members([-1], [3], [0], [4], 4, 1, 2) == ([0, 0, 0, -1], [2, 2, 2, 0])
    state = torch.tensor([0, 2, 0, 0, 1, 3], dtype=torch.int32)
    table = torch.tensor([[4, 1, PAD], [5, 4, 2]], dtype=torch.int32)
    s, t, remap, source, hole = orc.compact(state, table, [0, 1], [3, 3], 9)
    assert source == [4, 5] and hole == [0, 2] and s.tolist() == [1, 2, 3, 0, 0, 0] and remap.tolist() == [-1, 1, -1, -1, 0, 2]
    assert t.tolist() == [[0, 1, PAD], [2, 0, 2]]
    s, freed, wrong = orc.release(torch.tensor([[0, 1, 7], [0, 0, 0]]), [0, 1], [3, 2], 9, torch.tensor([2, 1]))
    assert (s.tolist(), freed, wrong) == ([0, 0], 2, 2)


# ------------------------------------------------------------------------------------------------ inputs
def _rows(shape, g, dtype):
    x = torch.randn(shape, generator=g)
    return (x * torch.exp(0.7 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)


def _case(seed, Hq, Hkv, D, dtype, groups, alone=(), slots_more=17):
    """groups: (prefix, [own tokens of the members]); alone: own tokens of the requests behind them.  Every group's prefix is named by a row of its own; the members' own rows
    hold nothing there."""
    g = torch.Generator().manual_seed(seed)
    B = sum(len(o) for _, o in groups) + len(alone)
    own = [n for _, o in groups for n in o] + list(alone)
    pre = [p for p, o in groups for _ in o] + [0] * len(alone)
    R = B + len(groups) + 2
    slots = sum(p for p, _ in groups) + sum(own) + slots_more
    perm = torch.randperm(slots, generator=g).to(torch.int32)
    rows = torch.randperm(R, generator=g).to(torch.int32)
    table = torch.full((R, max([p + n for p, n in zip(pre, own)] + [p for p, _ in groups] + [1]) + 3), PAD, dtype=torch.int32)
    at = 0
    for i, (p, _) in enumerate(groups):
        table[int(rows[B + i]), :p] = perm[at:at + p]
        at += p
    for b in range(B):
        table[int(rows[b]), pre[b]:pre[b] + own[b]] = perm[at:at + own[b]]
        at += own[b]
    starts, sizes, s = [], [], 0
    for _, o in groups:
        starts.append(s)
        sizes.append(len(o))
        s += len(o)
    return dict(q=_rows((B, Hq, D), g, dtype), kv=_rows((slots, 2 * Hkv, D), g, dtype), table=table, req=rows[:B].clone(),
                len=torch.tensor([p + n for p, n in zip(pre, own)], dtype=torch.int32), g=(starts, sizes, rows[B:B + len(groups)].tolist(), [p for p, _ in groups]),
                most=max([p for p, _ in groups] + [0]), own=max(own + [0]), Hkv=Hkv)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _decode_on_gpu(lsa, c, **kw):
    kv = c.get("kv_gpu", c["kv"].to(DEV))
    k, v = kv[:, :c["Hkv"]], kv[:, c["Hkv"]:]
    most = kw.pop("most", c["most"])
    return lsa.longserve_shared_prefix_decode_attention(c["q"].to(DEV), c["table"].to(DEV), c["req"].to(DEV), c["len"].to(DEV), int(c["len"].max()) if len(c["len"]) else 0,
                                                        k, v, *(_i32(x) for x in c["g"]), most, max_own_len=c["own"], **kw)


def _check(got, want, what):
    (o, lse), (o_ref, l_ref, tol_o, tol_l) = got, want
    o, lse = o.double().cpu(), lse.double().cpu()
    dead = torch.isneginf(l_ref)
    assert torch.equal(torch.isneginf(lse), dead), what
    assert bool((o[dead] == 0).all()), what
    off = ((o - o_ref).abs() / tol_o.clamp(min=1e-300))[~dead]
    assert not len(off) or float(off.max()) <= 1, (what, float(off.max()))
    off = ((lse - l_ref).abs() / tol_l.clamp(min=1e-300))[~dead]
    assert not len(off) or float(off.max()) <= 1, (what, "lse", float(off.max()))


def _decode_check(lsa, c, what, out_dtype=None, **kw):
    got = _decode_on_gpu(lsa, c, **kw)
    kv = c["kv"]
    _check(got, orc.decode(c["q"], kv[:, :c["Hkv"]], kv[:, c["Hkv"]:], c["table"], c["req"], c["len"], *c["g"], kw.get("most", c["most"]), out_dtype or c["q"].dtype), what)
    return got


GROUPS = {
    "one": ([(200, [1, 33, 64, 7])], []),
    "one-key": ([(1, [1, 2])], [5]),
    "tile-ends": ([(63, [3]), (64, [0, 5]), (65, [32, 31, 1]), (128, [1])], [1, 40]),
    "rows-past-a-tile": ([(130, [2] * 37)], [9, 1]),
    "long": ([(1000, [100] * 5), (513, [0] * 3)], []),
    "alone": ([], [1, 70, 300]),
    "no-own": ([(300, [0, 0, 0])], []),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(4, 4, 128), (8, 2, 128), (7, 1, 128), (20, 2, 64), (6, 6, 64), (16, 1, 128)])
@pytest.mark.parametrize("name", list(GROUPS))
def test_decode_against_float64(lsa, name, heads, dtype):
    groups, alone = GROUPS[name]
    _decode_check(lsa, _case(11, *heads, dtype, groups, alone), (name, heads, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_many_groups_and_a_large_batch(lsa, dtype):
    """More than 64 groups, more than 64 requests, and requests between the groups that none names."""
    c = _case(3, 4, 2, 64, dtype, [(5 + 3 * (i % 40), [i % 3, 1]) for i in range(140)], [3] * 30)
    _decode_check(lsa, c, "140 groups")
    # every second group dropped: its members (whose rows hold nothing in front) attend to their own tokens alone
    c["g"] = tuple(x[::2] for x in c["g"])
    _decode_check(lsa, c, "70 groups with gaps")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads, groups", [((64, 32, 64), [(2000, [1] * 150), (700, [0, 3] * 40)]), ((16, 2, 128), [(70, [9] * 17), (1300, [0, 40] * 20), (300, [2])]),
                                           ((128, 64, 64), [(1000, [0] * 130)]), ((32, 4, 64), [(60 + 37 * i, [i % 3] * (15 + i)) for i in range(12)])])
def test_decode_groups_of_several_row_tiles(lsa, heads, groups, dtype):
    """Row tiles that go through their group's prefix side by side, groups of one and of several; few workgroups per KV head and many."""
    _decode_check(lsa, _case(6, *heads, dtype, groups, [5, 900]), heads)


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [(32, 4, 64), (32, 8, 128), (128, 128, 128)])
def test_decode_large_batches(lsa, heads):
    """Rows enough to be joined by a wave each: from one partial to more than a wave has lanes, none among them."""
    groups = [(5, [0] * 3), (900, [3, 200, 0] * 8), (64, [33] * 50), (2500, [1] * 40)] if heads[0] < 100 else [(70, [1, 0, 500]), (1100, [2] * 20), (1, [0] * 12)]
    c = _case(8, *heads, torch.float16, groups, [0, 2100, 1] + [9] * 9)
    assert len(c["q"]) * heads[0] >= 4096
    _decode_check(lsa, c, heads)


@pytest.mark.gpu
def test_decode_lists_that_say_strange_things(lsa):
    """Overlapping groups, groups past the batch, unknown rows, negative numbers, a prefix past its bound: each as documented, none reads out of range."""
    c = _case(5, 8, 2, 128, torch.float16, [(100, [3, 4, 5]), (70, [1, 2])], [6, 2])
    full = c["table"].clone()
    s, n, r, p = c["g"]
    for b in range(5):  # the members' own rows name the prefixes too
        g = 0 if b < 3 else 1
        full[int(c["req"][b]), :p[g]] = full[r[g], :p[g]]
    c["table"] = full
    for what, g in (("overlap", ([0, 2], [3, 3], r, p)), ("past the batch", ([0, 3], [3, 99], r, p)), ("outside", ([0, 7], [3, 2], r, p)),
                    ("negative start", ([-2, 3], [3, 2], r, p)), ("negative size", (s, [3, -1], r, p)), ("unknown row", (s, n, [r[0], 999], p)),
                    ("negative row", (s, n, [-1, r[1]], p)), ("negative prefix", (s, n, r, [100, -5])), ("longer than its members", (s, n, r, [100, 72])),
                    ("none", ([], [], [], []))):
        c["g"] = g
        _decode_check(lsa, c, what)
    c["g"] = (s, n, r, p)
    _decode_check(lsa, c, "a prefix past the bound", most=64)
    _decode_check(lsa, c, "nobody shares", most=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_positions_that_do_not_exist(lsa, dtype):
    """Entries without a slot in prefixes and own rows, padded and short requests, NaN and infinities in every slot that is not named."""
    c = _case(7, 8, 2, 128, dtype, [(150, [3, 40, 0, 9]), (64, [2, 2])], [5, 0])
    t, (s, n, r, p) = c["table"], c["g"]
    t[r[0], 3], t[r[0], 70:100], t[r[0], 149] = PAD, -1, len(c["kv"])
    t[r[1], :64] = PAD  # nothing of the prefix exists
    t[int(c["req"][1]), 150:160] = PAD
    t[int(c["req"][4]), 64:66] = -7  # nothing at all
    c["len"][3] = 0    # a padded row of a group
    c["len"][0] = 100  # shorter than its prefix: alone, and its own row is empty there
    named = orc.valid(t.reshape(-1), len(c["kv"]))
    bad = torch.ones(len(c["kv"]), dtype=torch.bool)
    bad[named] = False
    assert bad.any()
    c["kv"][bad] = math.nan
    c["kv"][bad.nonzero()[::2, 0]] = math.inf
    if not bad[0]:  # slot 0, which is read in place of one that does not exist, is among them
        free = int(bad.nonzero()[0])
        c["kv"][[0, free]] = c["kv"][[free, 0]]
        c["table"] = torch.where(t == 0, free, t)
    _decode_check(lsa, c, "holes")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_maxima_that_rise_and_weights_far_apart(lsa, dtype):
    """Scores that rise by hundreds along the prefix, a first key that outweighs all others, equal scores; V up to the type's largest values."""
    for what in ("rise", "first", "equal", "large"):
        c = _case(9, 8, 2, 128, dtype, [(700, [5, 5, 5])], [40])
        slots = c["table"][c["g"][2][0], :700].long()
        k = c["kv"][:, :2]
        if what == "rise":
            k[slots] = (k[slots].float() * torch.linspace(0, 6, 700)[:, None, None]).to(dtype)
        if what == "first":
            k[slots[0]] = c["q"][0, ::4].float().mul(3).to(dtype)
        if what == "equal":
            k[:] = 0
        if what == "large":
            c["kv"][:, 2:] = (c["kv"][:, 2:].float().clamp(-1, 1) * (60000.0 if dtype == torch.float16 else 1e30)).to(dtype)
        _decode_check(lsa, c, what)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_decode_into_the_callers_tensors(lsa, out_dtype):
    """out of each type, the log-sum-exp and the workspace from the caller; strides of a pool with wider rows; what lies beside stays."""
    c = _case(13, 8, 2, 128, torch.float16, [(140, [1, 20, 3]), (90, [4])], [33])
    wide = torch.full((len(c["kv"]), 5, 160), math.nan, dtype=torch.float16)
    wide[:, :4, :128] = c["kv"]
    c["kv_gpu"] = wide.to(DEV)[:, :4, :128]
    B = len(c["q"])
    out, lse = torch.full((B + 2, 8, 128), 7.0, dtype=out_dtype, device=DEV), torch.full((B + 2, 8), 7.0, device=DEV)
    need = lsa.shared_prefix_decode_workspace_bytes(B, 2, 8, 2, 128, c["most"], c["own"])
    ws = torch.full((need + 64,), 77, dtype=torch.uint8, device=DEV)
    got = _decode_check(lsa, c, out_dtype, out_dtype=out_dtype, out=out[1:-1], o_logexpsum=lse[1:-1], workspace=ws[:need])
    assert got[0].data_ptr() == out[1].data_ptr() and got[1].data_ptr() == lse[1].data_ptr()
    assert bool((out[[0, -1]] == 7).all()) and bool((lse[[0, -1]] == 7).all()) and bool((ws[need:] == 77).all())
    for kw in (dict(workspace=ws[:need - 16]), dict(out=out[:B].double()), dict(out=out[:B - 1]), dict(o_logexpsum=lse[:B, :7]), dict(workspace=ws[::2])):
        with pytest.raises(ValueError):
            _decode_on_gpu(lsa, c, **kw)
    with pytest.raises(ValueError):
        _decode_on_gpu(lsa, dict(c, q=c["q"].bfloat16()))
    with pytest.raises(ValueError):
        _decode_on_gpu(lsa, c, most=-1)
    empty = dict(c, q=c["q"][:0], req=c["req"][:0], len=c["len"][:0], g=([], [], [], []))
    o, l = _decode_on_gpu(lsa, empty)
    assert o.shape == (0, 8, 128) and l.shape == (0, 8)


@pytest.mark.gpu
def test_decode_equals_decode_of_each_request(lsa):
    """The same requests through the operator that knows no groups (float32 out): as near as the weights' bits allow."""
    c = _case(17, 32, 8, 128, torch.float16, [(2000, [30] * 6)], [])
    t = c["table"]
    for b in range(6):
        t[int(c["req"][b]), :2000] = t[c["g"][2][0], :2000]
    o, lse = _decode_on_gpu(lsa, c, out=torch.empty(c["q"].shape, device=DEV))
    kv = c["kv"].to(DEV)
    ref_o, ref_l = lsa.longserve_window_decode_attention(c["q"].to(DEV), t.to(DEV), c["req"].to(DEV), c["len"].to(DEV), 2030, kv[:, :8], kv[:, 8:], 4000)
    # each weight off by 2^-11 at most, twice (numerator and sum), relative to the sum of |weight * V| <= the largest |V|
    assert float((o - ref_o).abs().max()) <= 2 * 2.0 ** -11 * float(kv[:, 8:].abs().max()) and float((lse - ref_l).abs().max()) <= 1e-5


# ------------------------------------------------------------------------------------------------ the prompts' step
def _prompt_case(seed, Hq, Hkv, D, dtype, groups, tail=3):
    """groups: (prefix, rows); `tail` rows of no group behind them."""
    g = torch.Generator().manual_seed(seed)
    T = sum(r for _, r in groups) + tail
    slots = sum(p for p, _ in groups) + 9
    perm = torch.randperm(slots, generator=g).to(torch.int32)
    rows = torch.randperm(len(groups) + 2, generator=g).tolist()
    table = torch.full((len(groups) + 2, max([p for p, _ in groups] + [1]) + 2), PAD, dtype=torch.int32)
    at, starts, s = 0, [], 0
    for i, (p, r) in enumerate(groups):
        table[rows[i], :p] = perm[at:at + p]
        at += p
        starts.append(s)
        s += r
    return dict(q=_rows((T, Hq, D), g, dtype), kv=_rows((slots, 2 * Hkv, D), g, dtype), table=table, g=(starts, [r for _, r in groups], rows[:len(groups)], [p for p, _ in groups]),
                most=max([p for p, _ in groups] + [1]), rows=max([r for _, r in groups] + [1]), Hkv=Hkv, gen=g)


def _prompt_on_gpu(lsa, c, o, m, l, **kw):
    kv = c["kv"].to(DEV)
    s, n, r, p = (_i32(x) for x in c["g"])
    lsa.shared_prefix_attention_fwd(c["q"].to(DEV) if "q_gpu" not in c else c["q_gpu"], kv[:, :c["Hkv"]], kv[:, c["Hkv"]:], o, s, n, c["table"].to(DEV), r, p, c["rows"],
                                    kw.pop("most", c["most"]), m, l, **kw)


def _prompt_ref(c, most=None):
    # (many rows: a bfloat16 V as fp16 and P in 11 bits for both types)
    q, kv = c["q"], c["kv"]
    return orc.prompt(q, kv[:, :c["Hkv"]], kv[:, c["Hkv"]:], c["table"], *c["g"], c["most"] if most is None else most, 2.0 ** -11)


PROMPTS = {
    "few": [(200, 3), (64, 10), (65, 1)],
    "one": [(1, 1)],
    "short-and-long": [(500, 40), (3, 90)],
    "none-in-one": [(70, 0), (129, 33), (0, 5)],
    "many": [(300, 700), (129, 500)],
    "many-one": [(1, 1500)],
    "twelve": [(40 + 61 * i, 5 + 29 * i) for i in range(12)],
    "prefill-kernel": [(70, 9000), (65, 5100)],
}
# rows and heads that hand the laid-out prefix to the prefill kernel (rows x heads of 98304 and more, a row per group and head of 512 and more)
WIDE = (128, 64, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (7, 1, 128)])
@pytest.mark.parametrize("name", list(PROMPTS))
def test_prompt_step_against_float64(lsa, name, heads, dtype):
    """From the empty state (o holds NaN) and, the second time, folded onto another step's state; rows of no group and without a key stay as they were."""
    c = _prompt_case(23, *heads, dtype, PROMPTS[name])
    T, Hq, D = c["q"].shape
    ref = _prompt_ref(c)
    o_ref, l_ref, tol_o, tol_l = ref
    dead = torch.isneginf(l_ref)
    o = torch.full((T, Hq, D), math.nan, dtype=dtype, device=DEV)
    m, l = torch.full((T, Hq), -math.inf, device=DEV), torch.zeros(T, Hq, device=DEV)
    _prompt_on_gpu(lsa, c, o, m, l)
    lse = (torch.log2(l) + m) * math.log(2)
    assert bool(torch.isnan(o.cpu()[dead]).all()) and bool((l.cpu()[dead] == 0).all()) and bool(torch.isneginf(m.cpu()[dead]).all())
    o[dead.to(DEV)] = 0
    _check((o, lse), (o_ref, l_ref, tol_o + orc.EPS_OUT[dtype] * (o_ref.abs() + tol_o) + 2.0 ** -25, tol_l + 1e-6), (name, heads, dtype))
    # folded: old state (o0, lse0) known exactly
    o0 = _rows((T, Hq, D), c["gen"], dtype)
    m0, l0 = torch.randn(T, Hq, generator=c["gen"]) + 2, torch.rand(T, Hq, generator=c["gen"]) * 3 + 0.5
    o, m, l = o0.to(DEV), m0.to(DEV), l0.to(DEV)
    _prompt_on_gpu(lsa, c, o, m, l)
    lse0 = (m0.double() + torch.log2(l0.double())) * math.log(2)
    both = torch.logaddexp(lse0, l_ref)
    w0, w1 = torch.exp(lse0 - both)[..., None], torch.exp(l_ref - both)[..., None]
    o_both = o0.double() * w0 + o_ref * w1
    # the weights follow the log-sum-exps: off by tol_l (and as much as float32's rounding of m, l), relatively
    err = tol_l[..., None] + 32 * orc.EPS32 * (1 + lse0.abs()[..., None] + both.abs()[..., None])
    tol = w1 * tol_o + err * (o0.double().abs() * w0 + o_ref.abs() * w1)
    tol = torch.where(dead[..., None], torch.zeros_like(tol), tol + orc.EPS_OUT[dtype] * (o_both.abs() + tol) + 2.0 ** -25)
    assert bool(((o.double().cpu() - o_both).abs() <= tol).all()), (name, heads, dtype)
    got = (torch.log2(l.double().cpu()) + m.double().cpu()) * math.log(2)
    assert bool(((got - both).abs() <= err[..., 0] + tol_l).all())
    assert torch.equal(m.cpu()[dead], m0[dead]) and torch.equal(l.cpu()[dead], l0[dead]) and torch.equal(o.cpu()[dead], o0[dead])


@pytest.mark.gpu
@pytest.mark.parametrize("heads, rows", [((8, 2, 128), 20), ((8, 2, 128), 800), (WIDE, 400), ((64, 2, 64), 790)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_step_entries_without_a_slot(lsa, heads, rows, dtype):
    """Holes in the prefix, prefixes cut at their bound, groups past q's rows, and NaN in every slot that is not named: both ways that the step is taken."""
    c = _prompt_case(29, *heads, dtype, [(200, rows), (90, rows), (80, 3)])
    t, (s, n, r, p) = c["table"], c["g"]
    t[r[0], :5], t[r[0], 63:66], t[r[0], 199] = PAD, -3, len(c["kv"]) + 4
    t[r[2], :80] = PAD
    named = orc.valid(t.reshape(-1), len(c["kv"]))
    bad = torch.ones(len(c["kv"]), dtype=torch.bool)
    bad[named] = False
    c["kv"][bad] = math.nan
    T, Hq, D = c["q"].shape
    for most, g in ((c["most"], c["g"]), (77, c["g"]), (c["most"], (s, [n[0], n[1] + 9999, n[2]], r, p)), (c["most"], ([-4, s[1], s[2]], n, [r[0], 99, r[2]], p))):
        c["g"] = g
        c["rows"] = min(max(g[1]), T)
        o_ref, l_ref, tol_o, tol_l = _prompt_ref(c, most)
        dead = torch.isneginf(l_ref)
        o, m, l = torch.zeros(T, Hq, D, dtype=dtype, device=DEV), torch.full((T, Hq), -math.inf, device=DEV), torch.zeros(T, Hq, device=DEV)
        _prompt_on_gpu(lsa, c, o, m, l, most=most)
        _check((o, (torch.log2(l) + m) * math.log(2)), (o_ref, l_ref, tol_o + orc.EPS_OUT[dtype] * (o_ref.abs() + tol_o) + 2.0 ** -25, tol_l + 1e-6), (heads, rows, most))


@pytest.mark.gpu
@pytest.mark.parametrize("heads, rows", [((8, 2, 128), 30), ((8, 2, 128), 900), (WIDE, 830)])
def test_prompts_behind_a_prefix_with_their_own_chunks(lsa, heads, rows):
    """The whole of a step: own chunks by context_attention_fwd, the prefix by shared_prefix_attention_fwd, in either order, on views with wider strides; against causal
    attention over prefix and chunk."""
    Hkv = heads[1]
    c = _prompt_case(31, *heads, torch.float16, [(333, rows)], tail=0)
    lens = [rows // 3, rows - rows // 3]
    T, Hq, D = c["q"].shape
    own = _rows((T, 2 * Hkv, D), c["gen"], torch.float16)
    slots = c["table"][c["g"][2][0], :333].long()
    want, looked_at = [], list(range(0, T, 1 if Hq < 100 else 37)) + [T - 1]
    for at, n in ((0, lens[0]), (lens[0], lens[1])):
        kk, vv = torch.cat([c["kv"][slots, :Hkv], own[at:at + n, :Hkv]]), torch.cat([c["kv"][slots, Hkv:], own[at:at + n, Hkv:]])
        for i in (x - at for x in looked_at if at <= x < at + n):
            want.append(orc.attend(c["q"][at + i:at + i + 1], kk[:333 + i + 1], vv[:333 + i + 1], 2.0 ** -11))
    o_ref, l_ref, tol_o, tol_l = (torch.cat(x) for x in zip(*want))
    q_wide = torch.zeros(T, Hq + 2, D, dtype=torch.float16, device=DEV)
    q_wide[:, 1:-1] = c["q"].to(DEV)
    c["q_gpu"] = q_wide[:, 1:-1]
    own_gpu = own.to(DEV)
    starts, n, zero = _i32([0, lens[0]]), _i32(lens), _i32([0, 0])
    for prefix_first in (True, False):
        o_wide = torch.full((T, Hq + 1, D), 3.0, dtype=torch.float16, device=DEV)
        ml = torch.zeros(2, T, Hq + 1, device=DEV)
        ml[0] = -math.inf
        o, m, l = o_wide[:, :Hq], ml[0, :, :Hq], ml[1, :, :Hq]
        if prefix_first:
            _prompt_on_gpu(lsa, c, o, m, l)
        lsa.context_attention_fwd(c["q_gpu"], own_gpu[:, :Hkv], own_gpu[:, Hkv:], o, starts, n, zero, starts, n, zero, 1, max(lens), m, l)
        if not prefix_first:
            _prompt_on_gpu(lsa, c, o, m, l)
        assert bool((o_wide[:, Hq] == 3).all()) and bool((ml[1, :, Hq] == 0).all())
        # o is rounded twice, by half a step of a value that is at most as large as |V|
        top = float(torch.cat([c["kv"][:, Hkv:].abs().amax()[None], own[:, Hkv:].abs().amax()[None]]).max())
        _check((o[looked_at], ((torch.log2(l) + m) * math.log(2))[looked_at]), (o_ref, l_ref, tol_o + 2 * 2.0 ** -11 * top, tol_l + 1e-5), prefix_first)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, prefix", [(64, 10253), (256, 2711), (8, 9000)])
def test_prompt_step_pieces_of_a_long_prefix(lsa, heads, prefix):
    """Row tiles that go through a long prefix side by side, in pieces: two and three of them per workgroup with few workgroups per head, one with many; every 29th row."""
    c = _prompt_case(33, heads, heads, 64, torch.float16, [(prefix, 300), (70, 2)], tail=0)
    T, Hq, D = c["q"].shape
    c["table"][c["g"][2][0], 100] = PAD
    rows = list(range(0, T, 29)) + [T - 1]
    of = [int(i >= 300) for i in rows]
    want = [_prompt_ref(dict(c, q=c["q"][i:i + 1], g=([0], [1], [c["g"][2][n]], [c["g"][3][n]]))) for i, n in zip(rows, of)]
    o_ref, l_ref, tol_o, tol_l = (torch.cat(x) for x in zip(*want))
    o, m, l = torch.zeros(T, Hq, D, dtype=torch.float16, device=DEV), torch.full((T, Hq), -math.inf, device=DEV), torch.zeros(T, Hq, device=DEV)
    _prompt_on_gpu(lsa, c, o, m, l)
    _check((o[rows], ((torch.log2(l) + m) * math.log(2))[rows]), (o_ref, l_ref, tol_o + 2.0 ** -11 * (o_ref.abs() + tol_o) + 2.0 ** -25, tol_l + 1e-6), (heads, prefix))


@pytest.mark.gpu
def test_prompt_step_refusals(lsa):
    c = _prompt_case(37, 8, 2, 128, torch.float16, [(20, 4)])
    T, Hq, D = c["q"].shape
    o, m, l = torch.zeros(T, Hq, D, dtype=torch.float16, device=DEV), torch.full((T, Hq), -math.inf, device=DEV), torch.zeros(T, Hq, device=DEV)
    before = o.clone(), m.clone(), l.clone()
    for bad in ((o.float(), m, l), (o[:-1], m, l), (o, m.half(), l), (o, m[:-1], l[:-1]), (o, m, l.t().contiguous().t())):
        with pytest.raises(ValueError):
            _prompt_on_gpu(lsa, c, *bad)
    with pytest.raises(ValueError):
        _prompt_on_gpu(lsa, c, o, m, l, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        _prompt_on_gpu(lsa, dict(c, kv=c["kv"].bfloat16()), o, m, l)
    _prompt_on_gpu(lsa, dict(c, g=([], [], [], [])), o, m, l)
    _prompt_on_gpu(lsa, c, o, m, l, most=0)
    assert all(torch.equal(a, b) for a, b in zip(before, (o, m, l)))


# ------------------------------------------------------------------------------------------------ forks, copies, releases
def _state_of(tables, size):
    state = torch.zeros(size, dtype=torch.int32)
    for s in tables.reshape(-1).tolist():
        if 0 <= s < size:
            state[s] += 1
    return state


@pytest.mark.gpu
@pytest.mark.parametrize("size, rows, width", [(50, 6, 9), (4000, 30, 700), (100000, 300, 300)])
def test_fork_and_release_against_lists(lsa, size, rows, width):
    g = torch.Generator().manual_seed(size)
    half = rows // 2
    table = torch.full((rows, width), PAD, dtype=torch.int32)
    lens = torch.randint(0, width + 1, (half,), generator=g).tolist()
    lens[0] = width
    for i, n in enumerate(lens):
        table[i, :n] = torch.randperm(size, generator=g)[:n].to(torch.int32)
    table[0, :2] = torch.tensor([-1, size])  # entries without a slot
    state = _state_of(table[:half], size)
    src = sorted(torch.randint(0, half, (rows - half,), generator=g).tolist())
    if size == 4000:
        src = [src[i] for i in torch.randperm(len(src), generator=g).tolist()]  # forks of one request here and there
    if size == 100000:
        src[:100] = [0] * 100  # a run of more than 64, the lengths rising
    flen = [min(lens[s], int(torch.randint(0, width + 50, (1,), generator=g))) for s in src]
    if size == 100000:
        flen[:100] = list(range(0, 300, 3))
    dst = [half + i for i in torch.randperm(rows - half, generator=g).tolist()]
    t, st = table.to(DEV), state.to(DEV)
    for most in (width, max(1, width // 2)):
        want_t, want_s = orc.fork(t.cpu(), src, dst, flen, most, st.cpu())
        lsa.fork_requests(t, _i32(src), _i32(dst), _i32(flen), most, st)
        assert torch.equal(t.cpu(), want_t) and torch.equal(st.cpu(), want_s)
    # all of them go, twice over: what is gone already, and what never was, is wrong and changes nothing
    req, rl = list(range(rows)) + [1, -1], lens + flen + [2, 3]
    want_s, freed, wrong = orc.release(t.cpu(), req, rl, width, st.cpu())
    got = st.clone()
    assert wrong > 0
    with pytest.raises(IndexError, match="%d tokens" % wrong):
        lsa.release_requests(t, _i32(req), _i32(rl), width, got)
    assert torch.equal(got.cpu(), want_s)
    ok = [i for i in range(half) if i != 0]
    want_s, freed, wrong = orc.release(t.cpu(), ok, [lens[i] for i in ok], width, st.cpu())
    assert wrong == 0 and lsa.release_requests(t, _i32(ok), _i32([lens[i] for i in ok]), width, st) == freed
    assert torch.equal(st.cpu(), want_s)
    assert lsa.release_requests(t, _i32([]), _i32([]), width, st) == 0 and lsa.release_requests(t, _i32([0]), _i32([5]), 0, st) == 0
    lsa.fork_requests(t, _i32([]), _i32([]), _i32([]), width, st)
    assert torch.equal(st.cpu(), want_s)


@pytest.mark.gpu
def test_release_of_one_slot_by_many(lsa):
    """Hundreds of requests hold the same few slots: each takes one reference, the last one frees; one more than there are is wrong."""
    table = torch.arange(20, dtype=torch.int32, device=DEV).repeat(500, 1).contiguous()
    for n in (150, 500):  # one workgroup, many
        state = torch.zeros(20, dtype=torch.int32, device=DEV)
        state[:19] = n
        state[5] = n + 1
        state[7] = n - 1
        with pytest.raises(IndexError, match="%d tokens" % (n + 1)):
            lsa.release_requests(table, torch.arange(n, dtype=torch.int32, device=DEV), _i32([20] * n), 20, state)
        want = torch.zeros(20, dtype=torch.int32)
        want[5] = 1
        assert torch.equal(state.cpu(), want)


def _raw_pool(g, layers, slots, heads, D, dtype):
    n = layers * slots * heads * D * (1 if dtype == F8 else 2)
    return torch.randint(0, 256, (n,), dtype=torch.uint8, generator=g).view(dtype).view(layers, slots, heads, D)


POOLS = [(1, 2, 64, F8), (3, 4, 128, torch.float16), (2, 16, 128, F8), (5, 2, 64, torch.bfloat16), (2, 64, 128, torch.float16), (1, 10, 64, F8)]


@pytest.mark.gpu
@pytest.mark.parametrize("layers, heads, D, dtype", POOLS)
def test_copies_bit_for_bit(lsa, layers, heads, D, dtype):
    g = torch.Generator().manual_seed(layers * heads)
    slots, width = 300, 60
    pool = _raw_pool(g, layers, slots + 5, heads, D, dtype)
    scales = torch.randint(0, 256, (layers, slots + 5, heads), dtype=torch.uint8, generator=g) if dtype == F8 else None
    perm = torch.randperm(slots, generator=g)
    table = torch.full((8, width), PAD, dtype=torch.int32)
    table[2, :width], table[5, :17] = perm[:60].to(torch.int32), perm[60:77].to(torch.int32)
    table[2, 4] = PAD
    src, dst, lens = [2, 5, 2, 5], [0, 7, 3, 1], [60, 17, 33, 0]
    index = perm[100:100 + sum(lens)].clone()
    start = [0, 60, 77, 110]
    want, want_t, want_sc = pool.view(torch.uint8).clone(), table.clone(), None if scales is None else scales.clone()
    for a, b, n, s in zip(src, dst, lens, start):
        for i in range(n):
            old, new = int(table[a, i]), int(index[s + i])
            want_t[b, i] = new
            if old != PAD:
                want[:, new] = pool.view(torch.uint8)[:, old]
                if scales is not None:
                    want_sc[:, new] = scales[:, old]
    p, t, sc = pool.to(DEV), table.to(DEV), None if scales is None else scales.to(DEV)
    lsa.copy_requests(t, _i32(src), _i32(dst), _i32(lens), _i32(start), width, index.to(DEV), p, sc)
    assert torch.equal(p.view(torch.uint8).cpu(), want) and torch.equal(t.cpu(), want_t) and (sc is None or torch.equal(sc.cpu(), want_sc))
    with pytest.raises(ValueError):
        lsa.copy_requests(t, _i32(src), _i32(dst), _i32(lens), _i32(start), width, index.to(DEV), p, None if sc is not None else torch.zeros(layers, slots + 5, heads, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError):
        lsa.copy_requests(t, _i32(src), _i32(dst), _i32(lens), _i32(start), width, index.to(DEV).int(), p, sc)
    with pytest.raises(ValueError):
        lsa.copy_requests(t, _i32(src), _i32(dst[:-1]), _i32(lens), _i32(start), width, index.to(DEV), p, sc)
    # an index that is too short, and slots outside the pool: those tokens are left out
    short = index[:70].clone()
    short[3] = slots + 5
    t2, p2 = table.to(DEV), pool.to(DEV)
    lsa.copy_requests(t2, _i32(src), _i32(dst), _i32(lens), _i32(start), width, short.to(DEV), p2, None if sc is None else scales.to(DEV))
    want_t2 = table.clone()
    for a, b, n, s in zip(src, dst, lens, start):
        for i in range(n):
            if s + i < 70 and (s + i) != 3:
                want_t2[b, i] = index[s + i]
    assert torch.equal(t2.cpu(), want_t2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, F8])
def test_copies_of_a_source_side_by_side(lsa, dtype):
    """Runs of forks of one source, one of more than 64, with lengths that rise and fall in them, sources and destinations that do not exist between them."""
    g = torch.Generator().manual_seed(9)
    layers, slots, width, n = 2, 9000, 130, 93
    pool = _raw_pool(g, layers, slots, 2, 32, dtype)
    scales = torch.randint(0, 256, (layers, slots, 2), dtype=torch.uint8, generator=g) if dtype == F8 else None
    src = [3] * 7 + [1] + [3] * 3 + [-1, 200] + [5] * 71 + [1] * 8 + [3]
    assert len(src) == n
    dst = list(range(10, 10 + n))
    dst[2], dst[40] = -7, 10 ** 6
    lens = torch.randint(0, width + 20, (n,), generator=g).tolist()
    lens[1], lens[50] = 0, -3
    table = torch.full((10 + n, width), PAD, dtype=torch.int32)
    table[:10] = torch.randint(0, 500, (10, width), generator=g).to(torch.int32)
    table[5, 7], table[3, 129] = -2, slots
    start = torch.tensor([0] + [max(0, min(x, width)) for x in lens]).cumsum(0)[:-1].tolist()
    index = torch.randperm(slots - 500, generator=g)[:start[-1] + width] + 500
    index[start[20]] = slots + 1
    want, want_t, want_sc = pool.view(torch.uint8).clone(), table.clone(), None if scales is None else scales.clone()
    for a, b, m, s in zip(src, dst, lens, start):
        if 0 <= a < 10 + n and 0 <= b < 10 + n:
            for i in range(min(m, width)):
                old, new = int(table[a, i]), int(index[s + i])
                if new < slots:
                    want_t[b, i] = new
                    if 0 <= old < slots:
                        want[:, new] = pool.view(torch.uint8)[:, old]
                        if scales is not None:
                            want_sc[:, new] = scales[:, old]
    p, t, sc = pool.to(DEV), table.to(DEV), None if scales is None else scales.to(DEV)
    lsa.copy_requests(t, _i32(src), _i32(dst), _i32(lens), _i32(start), width, index.to(DEV), p, sc)
    assert torch.equal(p.view(torch.uint8).cpu(), want) and torch.equal(t.cpu(), want_t) and (sc is None or torch.equal(sc.cpu(), want_sc))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1, 5, 300, 4096, 4097, 20000])
@pytest.mark.parametrize("share", [0.0, 0.03, 0.5, 0.97, 1.0])
@pytest.mark.parametrize("layers, heads, D, dtype", POOLS[:3])
def test_compaction_against_lists(lsa, size, share, layers, heads, D, dtype):
    g = torch.Generator().manual_seed(size + int(share * 100))
    idle = 3
    state = (torch.rand(size, generator=g) < share).int() * torch.randint(1, 4, (size,), generator=g).int()
    if size > 300:
        layers, heads = 1, 2
    pool = _raw_pool(g, layers, size + idle, heads, D, dtype)
    scales = torch.randint(0, 256, (layers, size + idle, heads), dtype=torch.uint8, generator=g) if dtype == F8 else None
    used = state.nonzero().squeeze(1)
    table = torch.full((4, 40), PAD, dtype=torch.int32)
    lens = [40, 13, 0]
    for i, n in enumerate(lens):
        if len(used):
            table[i, :n] = used[torch.randint(0, len(used), (n,), generator=g)].int()
    table[0, 7], table[1, 2] = PAD, -4
    if len(used) < size:
        table[0, 9] = int((state == 0).nonzero()[0])  # a free slot
    table[3, :5] = torch.arange(5)  # no live request: stays
    want_s, want_t, want_r, source, hole = orc.compact(state, table, [0, 1, 2], lens, 38)
    want = pool.view(torch.uint8).clone()
    want[:, hole] = want[:, source]
    st, t, p, sc = state.to(DEV), table.to(DEV), pool.to(DEV), None if scales is None else scales.to(DEV)
    remap = lsa.compact_pool(st, p, t, _i32([0, 1, 2]), _i32(lens), 38, sc)
    assert torch.equal(st.cpu(), want_s) and torch.equal(remap.cpu(), want_r) and torch.equal(t.cpu(), want_t) and torch.equal(p.view(torch.uint8).cpu(), want)
    if scales is not None:
        scales[:, hole] = scales[:, source]
        assert torch.equal(sc.cpu(), scales)
    # nothing moves the second time
    again = lsa.compact_pool(st, p, t, _i32([]), _i32([]), 0, sc, remap=torch.empty(size, dtype=torch.int32, device=DEV))
    n = int((state != 0).sum())
    assert torch.equal(again.cpu()[:n], torch.arange(n, dtype=torch.int32)) and bool((again.cpu()[n:] == -1).all())
    assert torch.equal(st.cpu(), want_s) and torch.equal(p.view(torch.uint8).cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [65536, 65537, 200001])
@pytest.mark.parametrize("share", [0.002, 0.6, 1.0])
def test_compaction_of_a_large_pool(lsa, size, share):
    """Pools whose counts come from a launch of their own, and the largest whose do not."""
    test_compaction_against_lists(lsa, size, share, 1, 2, 64, F8)


@pytest.mark.gpu
def test_compaction_refusals(lsa):
    st, p, t = torch.zeros(8, dtype=torch.int32, device=DEV), torch.zeros(2, 8, 2, 64, dtype=torch.float16, device=DEV), torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    i = _i32([0])
    for call in (lambda: lsa.compact_pool(st.long(), p, t, i, i, 4), lambda: lsa.compact_pool(st, p[:, :7], t, i, i, 4), lambda: lsa.compact_pool(st, p[0], t, i, i, 4),
                 lambda: lsa.compact_pool(st, p, t.long(), i, i, 4), lambda: lsa.compact_pool(st, p, t, i, _i32([0, 1]), 4), lambda: lsa.compact_pool(st, p, t, i, i, -1),
                 lambda: lsa.compact_pool(st, p, t, i, i, 4, torch.zeros(2, 8, 2, dtype=torch.uint8, device=DEV)),
                 lambda: lsa.compact_pool(st, p, t, i, i, 4, remap=torch.zeros(7, dtype=torch.int32, device=DEV)),
                 lambda: lsa.compact_pool(st, p, t, i, i, 4, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV)),
                 lambda: lsa.compact_pool(st, p.transpose(2, 3), t, i, i, 4)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.gpu
def test_a_search_from_its_first_prompt_to_its_end(lsa):
    """The managers and the attention as a serving program uses them: a prompt, forks of it that go on by themselves, decode steps over the shared prefix, some
    branches freed and one copied, the pool compacted under way, everything freed."""
    Hq, Hkv, D, layers = 8, 2, 128, 2
    mem = lsa.LongServeMemoryManager(600, torch.float16, Hkv, D, layers, num_idle_slots=2)
    reqs = lsa.LongServeReqManager(16, 200, mem)
    g = torch.Generator().manual_seed(1)
    mem.kv_buffer.copy_(torch.randn(mem.kv_buffer.shape, generator=g))
    noise = mem.alloc(100)
    parent = reqs.alloc(1)
    slots = mem.alloc(150)
    mem.free(noise[::2].contiguous())  # holes in front
    lsa.init_req_to_token_indexes(reqs.req_to_token_indexs, parent.int(), _i32([150]), slots)
    forks = reqs.fork(parent.repeat(5), _i32([150] * 5), 150)
    assert forks.tolist() == [1, 2, 3, 4, 5] and mem.mem_state[slots].unique().tolist() == [6]
    assert mem.can_use_mem_size == int((mem.mem_state == 0).sum()) and reqs.can_use_req_size == 10

    def attend(live, lens, layer):
        q = torch.randn(len(live), Hq, D, generator=torch.Generator().manual_seed(len(live) + layer)).half()
        cache = mem.kv_buffer[layer]
        ln = _i32(lens)
        o, lse = lsa.longserve_shared_prefix_decode_attention(q.to(DEV), reqs.req_to_token_indexs, live.int(), ln, max(lens), cache[:, :Hkv], cache[:, Hkv:], _i32([0]),
                                                              _i32([len(live)]), parent.int(), _i32([150]), 150)
        kv = cache.cpu()
        want = orc.decode(q, kv[:, :Hkv], kv[:, Hkv:], reqs.req_to_token_indexs.cpu(), live.cpu(), ln.cpu(), [0], [0], [0], [0], 0, torch.float16)  # each on its own
        _check((o, lse), want, lens)
        return o, lse

    lens = [150] * 5
    for step in range(4):
        new = mem.alloc(5)
        lens = [n + 1 for n in lens]
        lsa.copy_kv_index_to_req(reqs.req_to_token_indexs, forks.int(), _i32(lens), new)
        mem.kv_buffer[:, new] = torch.randn(layers, 5, 2 * Hkv, D, generator=g).half().to(DEV)
        for layer in range(layers):
            attend(forks, lens, layer)
    # two branches end; the prompt's slots keep the others' references
    reqs.free_reqs(forks[:2], _i32(lens[:2]), 154)
    assert mem.mem_state[slots].unique().tolist() == [4] and mem.can_use_mem_size == int((mem.mem_state == 0).sum())
    live = forks[2:]
    before = [attend(live, lens[2:], layer) for layer in range(layers)]
    used = 600 - mem.can_use_mem_size
    remap = mem.compact(reqs.req_to_token_indexs, torch.cat([parent, live]), _i32([150] + lens[2:]), 154)
    assert bool((mem.mem_state[:used] > 0).all()) and not bool(mem.mem_state[used:].any()) and mem.can_use_mem_size == 600 - used
    after = [attend(live, lens[2:], layer) for layer in range(layers)]
    assert all(torch.equal(a, b) for x, y in zip(before, after) for a, b in zip(x, y))  # the same rows in the same order
    noise = remap[noise[1::2]].long()
    slots = remap[slots].long()
    # a branch with copies of everything: its own slots, the same answers
    copy, own = reqs.fork_copy(live[:1], _i32(lens[2:3]), 154, 154)
    table = reqs.req_to_token_indexs
    assert torch.equal(table[int(copy[0]), :154].long(), own) and torch.equal(mem.kv_buffer[:, own], mem.kv_buffer[:, table[int(live[0]), :154].long()])
    assert mem.alloc_contiguous(600 - used - 154 - 1) is not None
    # the end
    everyone = torch.cat([parent, live, copy])
    reqs.free_reqs(everyone, _i32([150] + lens[2:] + [154]), 154)
    assert not bool(mem.mem_state[slots].any()) and not bool(mem.mem_state[own].any()) and int((mem.mem_state[noise] > 0).sum()) == 50
    assert reqs.can_use_req_size == 16 and mem.can_use_mem_size == int((mem.mem_state == 0).sum())
    assert reqs.fork(torch.zeros(17, dtype=torch.int32, device=DEV), _i32([1] * 17), 1) is None  # the table is full
    assert reqs.fork_copy(torch.zeros(17, dtype=torch.int32, device=DEV), _i32([1] * 17), 1, 17) is None
    with pytest.raises(IndexError):
        reqs.free_reqs(parent, _i32([150]), 150)


@pytest.mark.gpu
def test_captured_and_replayed(lsa):
    """Both attention operators, fork and compaction in one graph, replayed on changed inputs, eager work between the replays; each replay equals the eager call."""
    c = _case(41, 8, 2, 128, torch.float16, [(300, [4, 5, 6]), (70, [1, 20])], [3])
    pc = _prompt_case(43, 8, 2, 128, torch.float16, [(200, 25), (64, 4)])
    kv, q, t, req, ln = c["kv"].to(DEV), c["q"].to(DEV), c["table"].to(DEV), c["req"].to(DEV), c["len"].to(DEV)
    g = [_i32(x) for x in c["g"]]
    pkv, pq, pt, pg = pc["kv"].to(DEV), pc["q"].to(DEV), pc["table"].to(DEV), [_i32(x) for x in pc["g"]]
    T, Hq, D = pq.shape
    ws = torch.empty(lsa.shared_prefix_decode_workspace_bytes(len(q), 2, 8, 2, 128, 300, 20), dtype=torch.uint8, device=DEV)
    pws = torch.empty(lsa.shared_prefix_attention_workspace_bytes(T, 2, 8, 2, 128, 200), dtype=torch.uint8, device=DEV)
    o, lse = torch.empty_like(q), torch.empty(len(q), 8, device=DEV)
    po, m, l = torch.empty_like(pq), torch.empty(T, Hq, device=DEV), torch.empty(T, Hq, device=DEV)
    state, pool, table = torch.zeros(500, dtype=torch.int32, device=DEV), torch.randn(2, 500, 4, 64, device=DEV).half(), torch.full((6, 30), PAD, dtype=torch.int32, device=DEV)
    remap, cws = torch.empty_like(state), torch.empty(lsa.compact_workspace_bytes(500), dtype=torch.uint8, device=DEV)
    one, two, thirty = _i32([0, 0]), _i32([2, 3]), _i32([30, 11])

    def work():
        lsa.longserve_shared_prefix_decode_attention(q, t, req, ln, 306, kv[:, :2], kv[:, 2:], *g, 300, out=o, o_logexpsum=lse, workspace=ws, max_own_len=20)
        m.fill_(-math.inf)
        l.zero_()
        lsa.shared_prefix_attention_fwd(pq, pkv[:, :2], pkv[:, 2:], po, pg[0], pg[1], pt, pg[2], pg[3], 25, 200, m, l, workspace=pws)
        lsa.fork_requests(table, one, two, thirty, 30, state)
        lsa.compact_pool(state, pool, table, _i3, _l3, 30, remap=remap, workspace=cws)

    _i3, _l3 = _i32([0, 2, 3]), _i32([30, 30, 11])

    def reset(seed):
        r = torch.Generator().manual_seed(seed)
        q.copy_(torch.randn(q.shape, generator=r))
        pq.copy_(torch.randn(pq.shape, generator=r))
        state.zero_()
        table.fill_(PAD)
        slots = torch.randperm(500, generator=r)[:30].int().to(DEV)
        table[0, :30] = slots
        state[slots.long()] = 1
        pool.copy_(torch.randn(pool.shape, generator=r))

    outs = lambda: [x.clone() for x in (o, lse, po[:29], m[:29], l[:29], state, pool, table, remap)]  # noqa: E731
    want = []
    for seed in range(4):
        reset(seed)
        work()
        want.append(outs())
    reset(0)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work()
    for seed in (2, 0, 3, 1, 2):
        reset(seed)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs(), want[seed])), seed
        torch.mm(torch.randn(64, 64, device=DEV), torch.randn(64, 64, device=DEV)).sum().item()


@pytest.mark.gpu
def test_on_another_stream(lsa):
    """Calls go to the current stream: behind work that is queued there, and not in front of it."""
    c = _case(47, 8, 2, 128, torch.float16, [(400, [4, 5, 6])], [3])
    want = _decode_on_gpu(lsa, c)
    torch.cuda.synchronize()
    kv, kv2 = c["kv"].to(DEV), torch.zeros_like(c["kv"], device=DEV)
    c["kv_gpu"] = kv2
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        kv2.copy_(kv)
        got = _decode_on_gpu(lsa, c)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_slots_past_four_gigabytes(lsa):
    """Offsets of slots that need more than 32 bits, in attention, copies and compaction."""
    slots, Hkv, D = 1_300_000, 8, 128
    pool = torch.empty(1, slots, 2 * Hkv, D, dtype=torch.float16, device=DEV)
    g = torch.Generator().manual_seed(3)
    far = torch.tensor(sorted(torch.randperm(slots, generator=g)[:290].tolist() + list(range(slots - 10, slots))))
    rows = _rows((300, 2 * Hkv, D), g, torch.float16)
    pool[0, far.to(DEV)] = rows.to(DEV)
    table = torch.full((4, 300), PAD, dtype=torch.int32)
    small = table.clone()
    perm = torch.randperm(300, generator=g)
    for row, idx in ((0, perm[:200]), (1, perm[200:260]), (2, perm[260:300])):
        table[row, :len(idx)] = far[idx].int()
        small[row, :len(idx)] = idx.int()
    for row in (1, 2):  # behind the prefix
        for t in (table, small):
            t[row, 200:] = PAD
            n = 60 if row == 1 else 40
            t[row, 200:200 + n] = t[row, :n].clone()
    q = _rows((2, 16, D), g, torch.float16)
    gr = [_i32(x) for x in ([0], [2], [0], [200])]
    o, lse = lsa.longserve_shared_prefix_decode_attention(q.to(DEV), table.to(DEV), _i32([1, 2]), _i32([260, 240]), 260, pool[0, :, :Hkv], pool[0, :, Hkv:], *gr, 200)
    _check((o, lse), orc.decode(q, rows[:, :Hkv], rows[:, Hkv:], small, torch.tensor([1, 2]), torch.tensor([260, 240]), [0], [2], [0], [200], 200, torch.float16), "far")
    t = table.to(DEV)
    index = torch.arange(slots - 400, slots - 200, device=DEV)
    index = index[~torch.isin(index, far.to(DEV))][:100]
    lsa.copy_requests(t, _i32([0]), _i32([3]), _i32([100]), _i32([0]), 300, index, pool)
    assert torch.equal(pool[0, index].cpu(), rows[perm[:100]])
    state = torch.zeros(slots, dtype=torch.int32, device=DEV)
    state[far.to(DEV)] = 1
    remap = lsa.compact_pool(state, pool, t, _i32([0, 1, 2]), _i32([200, 300, 300]), 300)
    assert torch.equal(pool[0, t[0, :200].long()].cpu(), rows[perm[:200]]) and int(remap.max()) == 299 and bool(state[:300].all()) and not bool(state[300:].any())
