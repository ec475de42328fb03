"""Requests that share tokens of the KV pool: attention over shared prefixes, new requests over the slots of another (or over copies
of the rows), the release of requests' tokens, and compaction of the pool.  No reference counterparts: the reference's slots have
reference counts (loongserve/common/longserve_mem_manager.py:61-88), but nothing that makes requests share them.

A group of requests shares the slots of its first tokens.  Groups are four int32 vectors on the GPU:

  g_start_loc, g_size   the group's rows: requests of a decode batch, or rows of q of a prompts' step; groups in ascending order of their rows
  g_req_idx             the row of the request table that names the prefix (any member's, or one that is kept for it)
  g_prefix_len          how many of its first positions the group shares
"""
from __future__ import annotations

from operator import index as as_int
from typing import Optional, Tuple

import torch

from . import _lib, _native
from .ops import _i32vec, _on_current_device, _other_ints


def _table(t: torch.Tensor) -> None:
    if t.dtype != torch.int32 or t.dim() != 2 or not t.is_contiguous():
        raise ValueError("req_to_token_indexs must be a contiguous [max_req, max_seq] int32 tensor")


def _groups(start, size, req, prefix) -> None:
    n = start.shape[0]
    for t, name in ((start, "g_start_loc"), (size, "g_size"), (req, "g_req_idx"), (prefix, "g_prefix_len")):
        _i32vec(t, name, n)


def _pool_halves(q, cache_k, cache_v) -> None:
    if cache_k.dim() != 3 or cache_k.shape != cache_v.shape or cache_k.shape[2] != q.shape[2] or cache_k.dtype != q.dtype or cache_v.dtype != q.dtype:
        raise ValueError("cache_k and cache_v must be [slots, kv_heads, head_dim] of q's type and head_dim (an 8-bit pool: kv_gather_fp8 reads it back)")
    if cache_k.stride(2) != 1 or cache_v.stride(2) != 1:
        raise ValueError("cache_k and cache_v must be contiguous in head_dim")
    if q.shape[2] not in (64, 128):
        raise ValueError("head_dim must be 64 or 128 (got %d)" % q.shape[2])
    if cache_k.shape[1] == 0 or q.shape[1] == 0 or q.shape[1] % cache_k.shape[1]:
        raise ValueError("bad head counts: Hq=%d Hkv=%d" % (q.shape[1], cache_k.shape[1]))


def _workspace(workspace, need: int, what: str) -> None:
    if workspace is not None and (not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need):
        raise ValueError("workspace must be contiguous and hold at least %d bytes (%s)" % (need, what))


def shared_prefix_decode_workspace_bytes(batch_size: int, groups: int, q_head_num: int, kv_head_num: int, head_dim: int, max_prefix_len: int,
                                         max_own_len: int) -> int:
    """Bytes of device memory that longserve_shared_prefix_decode_attention needs for the partials of such a call, and of every call with the same heads in
    which no other size is larger."""
    return int(_lib.load().lsattn_shared_decode_workspace_bytes(int(batch_size), int(groups), int(q_head_num), int(kv_head_num), int(head_dim),
                                                                int(max_prefix_len), int(max_own_len)))


def longserve_shared_prefix_decode_attention(q: torch.Tensor, req_to_token_indexs: torch.Tensor, b_req_idx: torch.Tensor, b_seq_len: torch.Tensor,
                                             max_len_in_batch: int, cache_k: torch.Tensor, cache_v: torch.Tensor, g_start_loc: torch.Tensor,
                                             g_size: torch.Tensor, g_req_idx: torch.Tensor, g_prefix_len: torch.Tensor, max_prefix_len: int,
                                             out: Optional[torch.Tensor] = None, o_logexpsum: Optional[torch.Tensor] = None,
                                             workspace: Optional[torch.Tensor] = None, max_own_len: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Decode attention of one new token per request where groups of requests share their first tokens: (o, natural log-sum-exp).
    The prefix of a group is read and multiplied once for up to 128 query rows (requests times query heads of a KV head) together.

    q [batch, q_heads, head_dim] (float16 or bfloat16, head_dim 64 or 128), cache_k / cache_v the K and V heads of a pool of q's
    type (any slot and head strides that keep rows 16-byte aligned), b_seq_len whole lengths, prefixes included.  Group g are requests
    g_start_loc[g] .. + g_size[g] - 1 of the batch, in ascending order; its first g_prefix_len[g] tokens are the slots that row g_req_idx[g] of the table
    names.  A request of no group, or shorter than its group's prefix, attends by its own row of the table alone (a length of 0: o = 0,
    -inf), one that two groups name belongs to the first.  max_prefix_len bounds g_prefix_len: what a group has beyond it is read by each
    request for itself.  Entries of the table that name no slot count as positions that do not exist; a request whose own row is not in the table has none at all.

    out: q's type unless given (float16, bfloat16 or float32).  Over the prefixes a request's weights are rounded: to float16, 2^-11 of a weight, and o is divided by the sum
    of the rounded ones; or to two parts of bfloat16, 2^-16.  A float32 out, which lse_merge joins with another instance's, carries that.  The log-sum-exp is float32's.  max_len_in_batch, or max_own_len (a bound of the
    tokens behind the prefix) where given, only sizes the launch and weighs its two parts (a close bound helps).  workspace: the caller's scratch
    (shared_prefix_decode_workspace_bytes; else torch allocates it), one for each call that may run at the same time, graphs' replays among them."""
    own = max_len_in_batch if max_own_len is None else max_own_len
    done = _native.shared_decode(q, req_to_token_indexs, b_req_idx, b_seq_len, cache_k, cache_v, g_start_loc, g_size, g_req_idx, g_prefix_len,
                                 max_prefix_len, own, out, o_logexpsum, workspace)
    if done is not None:
        return done
    numbers = (max_len_in_batch, max_prefix_len, max_own_len)
    if _other_ints(*numbers):
        most, prefix, own = (None if x is None else as_int(x) for x in numbers)
        return longserve_shared_prefix_decode_attention(q, req_to_token_indexs, b_req_idx, b_seq_len, most, cache_k, cache_v, g_start_loc, g_size, g_req_idx,
                                                        g_prefix_len, prefix, out, o_logexpsum, workspace, own)
    # arguments the native pass does not take: say what is wrong
    _on_current_device(((q, "q"), (req_to_token_indexs, "req_to_token_indexs"), (b_req_idx, "b_req_idx"), (b_seq_len, "b_seq_len"), (cache_k, "cache_k"),
                        (cache_v, "cache_v"), (g_start_loc, "g_start_loc"), (g_size, "g_size"), (g_req_idx, "g_req_idx"), (g_prefix_len, "g_prefix_len"),
                        (out, "out"), (o_logexpsum, "o_logexpsum"), (workspace, "workspace")))
    if q.dtype not in (torch.float16, torch.bfloat16) or q.dim() != 3 or not q.is_contiguous():
        raise ValueError("q must be a contiguous float16 or bfloat16 [batch, heads, head_dim] tensor")
    B, Hq, D = q.shape
    _table(req_to_token_indexs)
    _i32vec(b_req_idx, "b_req_idx", B)
    _i32vec(b_seq_len, "b_seq_len", B)
    _groups(g_start_loc, g_size, g_req_idx, g_prefix_len)
    _pool_halves(q, cache_k, cache_v)
    if max_len_in_batch < 0 or max_prefix_len < 0 or (max_own_len is not None and max_own_len < 0):
        raise ValueError("max_len_in_batch, max_prefix_len and max_own_len must be >= 0")
    if out is not None and (out.dtype not in (torch.float16, torch.bfloat16, torch.float32) or out.shape != q.shape or not out.is_contiguous()):
        raise ValueError("out must be a contiguous float16, bfloat16 or float32 tensor of q's shape")
    if o_logexpsum is not None and (o_logexpsum.dtype != torch.float32 or tuple(o_logexpsum.shape) != (B, Hq) or not o_logexpsum.is_contiguous()):
        raise ValueError("o_logexpsum must be a contiguous float32 [batch, heads] tensor")
    _workspace(workspace, shared_prefix_decode_workspace_bytes(B, g_start_loc.shape[0], Hq, cache_k.shape[1], D, max_prefix_len, own),
               "shared_prefix_decode_workspace_bytes")
    if B == 0:
        return (torch.empty_like(q) if out is None else out,
                torch.empty((0, Hq), dtype=torch.float32, device=q.device) if o_logexpsum is None else o_logexpsum)
    raise ValueError("shared-prefix decode attention: arguments that no kernel takes (an empty pool?)")


def shared_prefix_attention_workspace_bytes(rows: int, groups: int, q_head_num: int, kv_head_num: int, head_dim: int, max_prefix_len: int) -> int:
    """Bytes of device memory that shared_prefix_attention_fwd needs for such a call.  They are enough for calls with the same heads and fewer rows, groups and
    shorter prefixes, too; calls with fewer groups may need more to have a prefix laid out and are taken without that where it is not there."""
    return int(_lib.load().lsattn_shared_prefill_workspace_bytes(int(rows), int(groups), int(q_head_num), int(kv_head_num), int(head_dim), int(max_prefix_len)))


def shared_prefix_attention_fwd(q: torch.Tensor, cache_k: torch.Tensor, cache_v: torch.Tensor, o: torch.Tensor, g_start_loc: torch.Tensor,
                                g_size: torch.Tensor, req_to_token_indexs: torch.Tensor, g_req_idx: torch.Tensor, g_prefix_len: torch.Tensor,
                                max_g_size: int, max_prefix_len: int, m: torch.Tensor, l: torch.Tensor,
                                workspace: Optional[torch.Tensor] = None) -> None:
    """The step of prompts' chunks over the prefix that they share, folded in place into (o, m, l) as context_attention_fwd folds a step;
    the requests' own chunks are steps of context_attention_fwd on the same (o, m, l), before or after.

    q, o [tokens, q_heads, head_dim] (float16 or bfloat16, head_dim 64 or 128, contiguous in head_dim), m, l float32 [tokens, q_heads] with the
    same strides.  Rows g_start_loc[g] .. + g_size[g] - 1 of q, the new tokens of all requests of group g, see all of the first g_prefix_len[g] tokens of row
    g_req_idx[g] of the table, whose K/V lie in the pool cache_k / cache_v ([slots, kv_heads, head_dim] of q's type).  Groups in ascending order of their rows; a
    row that two groups name belongs to the first; rows of no group stay as they are.  max_g_size and max_prefix_len bound g_size and
    g_prefix_len (rows past the one may stay uncomputed, prefixes are cut at the other).  Entries of the table that name no slot count as positions that
    do not exist.

    Few rows are multiplied with the pool's rows where they lie, their partials folded by a second launch; for many (98304 rows x heads, 512 rows x heads of a KV head per
    group) the prefix is laid out once for the kernel behind context_attention_fwd, with its precision: a bfloat16 V counts as float16 there (magnitudes past 65504 as 65504,
    below 2^-14 cut to multiples of 2^-24), the weights as float16.  Rows that come together in fewer calls or more may differ by so much.  workspace: the caller's scratch
    (shared_prefix_attention_workspace_bytes for q's rows; else torch allocates it), one for each call that may run at the same time."""
    if _native.shared_prefill(q, cache_k, cache_v, o, g_start_loc, g_size, req_to_token_indexs, g_req_idx, g_prefix_len, max_g_size, max_prefix_len, m, l,
                              workspace):
        return
    if _other_ints(max_g_size, max_prefix_len):
        return shared_prefix_attention_fwd(q, cache_k, cache_v, o, g_start_loc, g_size, req_to_token_indexs, g_req_idx, g_prefix_len, as_int(max_g_size),
                                           as_int(max_prefix_len), m, l, workspace)
    _on_current_device(((q, "q"), (cache_k, "cache_k"), (cache_v, "cache_v"), (o, "o"), (g_start_loc, "g_start_loc"), (g_size, "g_size"),
                        (req_to_token_indexs, "req_to_token_indexs"), (g_req_idx, "g_req_idx"), (g_prefix_len, "g_prefix_len"), (m, "m"), (l, "l"),
                        (workspace, "workspace")))
    if q.dtype not in (torch.float16, torch.bfloat16) or q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be a float16 or bfloat16 [tokens, heads, head_dim] tensor, contiguous in head_dim")
    if o.dtype != q.dtype or o.shape != q.shape or o.stride(2) != 1:
        raise ValueError("o must have the type and shape of q and be contiguous in head_dim")
    _table(req_to_token_indexs)
    _groups(g_start_loc, g_size, g_req_idx, g_prefix_len)
    _pool_halves(q, cache_k, cache_v)
    if m.dtype != torch.float32 or l.dtype != torch.float32 or m.shape != q.shape[:2] or l.shape != m.shape or m.stride() != l.stride():
        raise ValueError("m and l must be float32 [tokens, q_heads] with the same strides")
    if max_g_size < 0 or max_prefix_len < 0:
        raise ValueError("max_g_size and max_prefix_len must be >= 0")
    _workspace(workspace, shared_prefix_attention_workspace_bytes(q.shape[0], g_start_loc.shape[0], q.shape[1], cache_k.shape[1], q.shape[2],
                                                                  min(max_prefix_len, req_to_token_indexs.shape[1])), "shared_prefix_attention_workspace_bytes")
    if q.numel() == 0 or g_start_loc.shape[0] == 0 or max_g_size == 0 or max_prefix_len == 0:
        return
    raise ValueError("shared_prefix_attention_fwd: arguments that no kernel takes (an empty pool?)")


def fork_requests(req_to_token_indexs: torch.Tensor, src_req_idx: torch.Tensor, dst_req_idx: torch.Tensor, b_seq_len: torch.Tensor, max_len_in_batch: int,
                  mem_state: torch.Tensor) -> None:
    """New requests over the slots of others: row dst_req_idx[i] of the table gets the first b_seq_len[i] entries of row src_req_idx[i], and every slot in them one
    more reference in mem_state.  LongServeReqManager.fork does this with rows of its own.

    The index vectors and lengths are int32 on the GPU.  A source may be named any number of times (forks of one source next to each other cost one addition per
    token); destination rows are distinct and no source of the call.  Entries that name no slot are copied and not counted; positions of a source that is no row of the
    table, and those whose slot is free, name none in the new row (2147483647).  max_len_in_batch bounds b_seq_len: positions past it are left out."""
    if _native.fork_requests(req_to_token_indexs, src_req_idx, dst_req_idx, b_seq_len, max_len_in_batch, mem_state):
        return
    if _other_ints(max_len_in_batch):
        return fork_requests(req_to_token_indexs, src_req_idx, dst_req_idx, b_seq_len, as_int(max_len_in_batch), mem_state)
    _on_current_device(((req_to_token_indexs, "req_to_token_indexs"), (src_req_idx, "src_req_idx"), (dst_req_idx, "dst_req_idx"), (b_seq_len, "b_seq_len"),
                        (mem_state, "mem_state")))
    _table(req_to_token_indexs)
    n = src_req_idx.shape[0]
    for t, name in ((src_req_idx, "src_req_idx"), (dst_req_idx, "dst_req_idx"), (b_seq_len, "b_seq_len")):
        _i32vec(t, name, n)
    _i32vec(mem_state, "mem_state")
    if max_len_in_batch < 0:
        raise ValueError("max_len_in_batch must be >= 0")
    if n == 0 or max_len_in_batch == 0 or req_to_token_indexs.numel() == 0:
        return
    raise ValueError("fork_requests: arguments that no kernel takes (an empty pool?)")


def _rows_of(kv_buffer, kv_scales) -> None:
    if kv_buffer.dim() != 4 or kv_buffer.stride(3) != 1 or kv_buffer.stride(2) != kv_buffer.shape[3]:
        raise ValueError("kv_buffer must be [layers, slots, heads, head_dim] with contiguous rows")
    if (kv_scales is not None) != (kv_buffer.dtype == torch.float8_e4m3fn):
        raise ValueError("kv_scales belong to a float8_e4m3fn kv_buffer, and to no other")
    if kv_scales is not None and (kv_scales.dtype not in (torch.uint8, torch.float8_e8m0fnu) or kv_scales.shape != kv_buffer.shape[:3] or kv_scales.stride(2) != 1):
        raise ValueError("kv_scales must be uint8 (or float8_e8m0fnu) [layers, slots, heads], contiguous in the heads")


def copy_requests(req_to_token_indexs: torch.Tensor, src_req_idx: torch.Tensor, dst_req_idx: torch.Tensor, b_seq_len: torch.Tensor, b_start_loc: torch.Tensor,
                  max_len_in_batch: int, mem_index: torch.Tensor, kv_buffer: torch.Tensor, kv_scales: Optional[torch.Tensor] = None) -> None:
    """New requests over copies of others' tokens: the rows of the first b_seq_len[i] tokens of request src_req_idx[i] are copied, in every layer of kv_buffer ([layers, slots,
    heads, head_dim], any type; kv_scales are the exponents of an 8-bit one), to the slots mem_index[b_start_loc[i]:], which row dst_req_idx[i] of the table names
    then.  mem_index is what LongServeMemoryManager.alloc returns (int64), the index vectors and lengths are int32 on the GPU.  LongServeReqManager.fork_copy does
    this with rows and slots of its own.

    A source may be named any number of times; destination rows are distinct and no source of the call, slots of mem_index likewise.  A position whose entry in the source names
    no slot has its slot of mem_index like any other, whose K/V stay as they were: the caller's to write before the copy is attended to (fork_copy refuses such sources).  Positions
    for which mem_index has no slot of the pool (its end, a number outside) name none (2147483647), nor do those of a source that is no row of the table.
    max_len_in_batch bounds b_seq_len: positions past it are left out."""
    if _native.copy_requests(req_to_token_indexs, src_req_idx, dst_req_idx, b_seq_len, b_start_loc, max_len_in_batch, mem_index, kv_buffer, kv_scales):
        return
    if _other_ints(max_len_in_batch):
        return copy_requests(req_to_token_indexs, src_req_idx, dst_req_idx, b_seq_len, b_start_loc, as_int(max_len_in_batch), mem_index, kv_buffer, kv_scales)
    _on_current_device(((req_to_token_indexs, "req_to_token_indexs"), (src_req_idx, "src_req_idx"), (dst_req_idx, "dst_req_idx"), (b_seq_len, "b_seq_len"),
                        (b_start_loc, "b_start_loc"), (mem_index, "mem_index"), (kv_buffer, "kv_buffer"), (kv_scales, "kv_scales")))
    _table(req_to_token_indexs)
    n = src_req_idx.shape[0]
    for t, name in ((src_req_idx, "src_req_idx"), (dst_req_idx, "dst_req_idx"), (b_seq_len, "b_seq_len"), (b_start_loc, "b_start_loc")):
        _i32vec(t, name, n)
    if mem_index.dtype != torch.int64 or mem_index.dim() != 1 or not mem_index.is_contiguous():
        raise ValueError("mem_index must be a contiguous 1-D int64 tensor, as the allocator returns it")
    _rows_of(kv_buffer, kv_scales)
    if max_len_in_batch < 0:
        raise ValueError("max_len_in_batch must be >= 0")
    if n == 0 or max_len_in_batch == 0 or req_to_token_indexs.numel() == 0 or mem_index.numel() == 0 or kv_buffer.numel() == 0:
        return
    raise ValueError("copy_requests: arguments that no kernel takes")


def _sources_of_copies(req_to_token_indexs, src_req_idx, b_seq_len, max_len_in_batch, mem_state) -> Tuple[torch.Tensor, int, int]:
    """(the lengths as a copy takes them, their sum, how many of the positions have no slot, or one that is free).  Waits for the device."""
    _on_current_device(((req_to_token_indexs, "req_to_token_indexs"), (src_req_idx, "src_req_idx"), (b_seq_len, "b_seq_len")))
    _table(req_to_token_indexs)
    for t, name in ((src_req_idx, "src_req_idx"), (b_seq_len, "b_seq_len")):
        _i32vec(t, name, len(src_req_idx))
    if max_len_in_batch < 0:
        raise ValueError("max_len_in_batch must be >= 0")
    rows, width = req_to_token_indexs.shape
    most = min(as_int(max_len_in_batch), width)
    lens = b_seq_len.clamp(0, most)
    size = len(mem_state)
    if not len(src_req_idx) or not most or not rows or not size:
        return lens, 0, 0
    slots = req_to_token_indexs[src_req_idx.clamp(0, rows - 1), :most]
    there = (slots >= 0) & (slots < size) & (mem_state[slots.clamp(0, size - 1)] != 0) & ((src_req_idx >= 0) & (src_req_idx < rows))[:, None]
    missing = ~there & (torch.arange(most, device=slots.device) < lens[:, None])
    return lens, *torch.stack([lens.sum(), missing.sum()]).tolist()


def _release(req_to_token_indexs, b_req_idx, b_seq_len, max_len_in_batch, mem_state) -> Tuple[int, int]:
    counts = _native.release_requests(req_to_token_indexs, b_req_idx, b_seq_len, max_len_in_batch, mem_state)
    if counts is not None:
        return counts
    if _other_ints(max_len_in_batch):
        return _release(req_to_token_indexs, b_req_idx, b_seq_len, as_int(max_len_in_batch), mem_state)
    _on_current_device(((req_to_token_indexs, "req_to_token_indexs"), (b_req_idx, "b_req_idx"), (b_seq_len, "b_seq_len"), (mem_state, "mem_state")))
    _table(req_to_token_indexs)
    n = b_req_idx.shape[0]
    _i32vec(b_req_idx, "b_req_idx", n)
    _i32vec(b_seq_len, "b_seq_len", n)
    _i32vec(mem_state, "mem_state")
    if max_len_in_batch < 0:
        raise ValueError("max_len_in_batch must be >= 0")
    if n == 0 or max_len_in_batch == 0 or req_to_token_indexs.numel() == 0:
        return 0, 0
    raise ValueError("release_requests: arguments that no kernel takes (an empty pool?)")


def _check_released(wrong: int) -> None:
    if wrong:
        raise IndexError("%d tokens of the released requests name no slot of the pool, or one that was free already" % wrong)


def release_requests(req_to_token_indexs: torch.Tensor, b_req_idx: torch.Tensor, b_seq_len: torch.Tensor, max_len_in_batch: int, mem_state: torch.Tensor) -> int:
    """One reference less in mem_state on the slot of each of the first b_seq_len[i] tokens of the requests b_req_idx[i] (int32 on the GPU), for every request that
    holds it: requests that share tokens can be let go of in one call, where LongServeMemoryManager.free counts a slot that its list names twice once, as the reference's does.
    Returns how many slots became free (and so waits for the call).  The table stays as it is.  LongServeReqManager.free_reqs does this with its rows.

    max_len_in_batch bounds b_seq_len: positions past it are left out.  Tokens that name no slot, or one that is free already (its count stays 0), are an IndexError once
    everything else is released."""
    freed, wrong = _release(req_to_token_indexs, b_req_idx, b_seq_len, max_len_in_batch, mem_state)
    _check_released(wrong)
    return freed


def compact_pool(mem_state: torch.Tensor, kv_buffer: torch.Tensor, req_to_token_indexs: torch.Tensor, b_req_idx: torch.Tensor, b_seq_len: torch.Tensor,
                 max_len_in_batch: int, kv_scales: Optional[torch.Tensor] = None, remap: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Moves the slots in use to the front of the pool: with U of them (mem_state != 0), the k-th free slot below U takes the k-th used slot from U on, its row in every
    layer of kv_buffer ([layers, slots, heads, head_dim]; kv_scales are the exponents of an 8-bit one) and its count.  Behind it every free slot is one run, which
    alloc_contiguous finds.  The first b_seq_len[i] entries of the rows b_req_idx[i] of the table (the live requests) follow.

    Returns remap, int32 [pool size] (the caller's tensor, or a new one): where each used slot is now, -1 for a free one; whoever keeps slot numbers elsewhere takes
    remap[them].  Nothing waits for the device.  Slots of kv_buffer past mem_state's size (idle ones) stay.  max_len_in_batch bounds b_seq_len: entries past it stay as
    they are.  workspace: the caller's scratch (compact_workspace_bytes of the size), else torch allocates it."""
    given = remap
    if remap is None:
        remap = torch.empty_like(mem_state)
    if _native.compact_pool(mem_state, kv_buffer, req_to_token_indexs, b_req_idx, b_seq_len, max_len_in_batch, kv_scales, remap, workspace):
        return remap
    if _other_ints(max_len_in_batch):
        return compact_pool(mem_state, kv_buffer, req_to_token_indexs, b_req_idx, b_seq_len, as_int(max_len_in_batch), kv_scales, given, workspace)
    _on_current_device(((mem_state, "mem_state"), (kv_buffer, "kv_buffer"), (req_to_token_indexs, "req_to_token_indexs"), (b_req_idx, "b_req_idx"),
                        (b_seq_len, "b_seq_len"), (kv_scales, "kv_scales"), (remap, "remap"), (workspace, "workspace")))
    _i32vec(mem_state, "mem_state")
    _i32vec(remap, "remap", mem_state.shape[0])
    _rows_of(kv_buffer, kv_scales)
    if kv_buffer.shape[1] < mem_state.shape[0]:
        raise ValueError("kv_buffer must have a row for every slot of mem_state")
    _table(req_to_token_indexs)
    _i32vec(b_req_idx, "b_req_idx")
    _i32vec(b_seq_len, "b_seq_len", b_req_idx.shape[0])
    if max_len_in_batch < 0:
        raise ValueError("max_len_in_batch must be >= 0")
    _workspace(workspace, compact_workspace_bytes(mem_state.shape[0]), "compact_workspace_bytes")
    if mem_state.shape[0] == 0:
        return remap
    raise ValueError("compact_pool: arguments that no kernel takes")


def compact_workspace_bytes(pool_size: int) -> int:
    """Bytes of device memory that compact_pool needs for a pool of so many slots."""
    return int(_lib.load().lsattn_compact_workspace_bytes(int(pool_size)))
