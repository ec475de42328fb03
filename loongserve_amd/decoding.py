"""Python wrappers the llama layer calls for decode; names and argument order of
loongserve/models/llama/triton_kernel/longserve_flash_decoding_stage1.py:78,
longserve_flash_decoding_stage2.py:53 and longserve_flash_decoding.py:3."""
from __future__ import annotations

import functools
from operator import index as as_int
from typing import Optional, Tuple

import torch

from . import _lib, _native, longserve_cuda_kernels
from .ops import _fp8_pool, _i32vec, _on_current_device, _other_ints


# The stage functions called on their own (the master path, longserve_transformer_layer_infer.py:272-281 then :360-367)
# leave the reference's buffers: one partial per block of block_seq tokens, row i of mid_out = block i.
# Opt-in (STAGE1_MERGES_BLOCKS = True; not the reference's layout): stage 1 computes one partial per group of consecutive
# blocks (the same rule as the fused call below, at most 16 blocks), writes it to the row of the group's first block and
# marks the rows of the others empty (LSE = -inf, mid_out row left as it was).  Any LSE merge over ceil(len / block_seq)
# rows per request that skips empty rows (this package's stage 2 does) gives the same result, with a quarter of the
# partial bytes at BLOCK_SEQ 256; a consumer that multiplies an empty row's mid_out by a zero weight instead must not use
# it (the stale row may hold anything).
STAGE1_MERGES_BLOCKS = False


def longserve_flash_decode_stage1(q, k, v, Req_to_tokens, B_req_idx, B_Seqlen, max_len_in_batch, mid_out,
                                  mid_out_logsumexp, block_seq):
    merge = 1
    if STAGE1_MERGES_BLOCKS:
        merge = min(16, _fused_block_seq(block_seq, q.shape[0], max_len_in_batch, k.shape[1]) // int(block_seq))
    longserve_cuda_kernels.flash_decoding_stage1(mid_out, mid_out_logsumexp, q, k, v, Req_to_tokens, B_req_idx,
                                                 B_Seqlen, max_len_in_batch, block_seq, merge)
    return


def longserve_flash_decode_stage2(mid_out, mid_out_logexpsum, B_Seqlen, O, out_logexpsum, block_seq, lead_rows=0):
    longserve_cuda_kernels.flash_decoding_stage2(O, out_logexpsum, B_Seqlen, mid_out, mid_out_logexpsum, block_seq, lead_rows)
    return


# Split size between the two stages of the fused call.  There mid_o / mid_o_logexpsum are scratch (FDPY:12-27 never hands
# them out, the callers at longserve_transformer_layer_infer.py:293-308 only use the returned pair), so the context may be
# cut more coarsely than BLOCK_SEQ: fewer fp32 block partials are written while the gather saturates the memory system
# (every MB of them costs about as much as 8 MB of reads).  The result is the same softmax, merged from fewer pieces.
# longserve_flash_decode_stage1 / _stage2 called on their own always split at the block_seq they are given.
# (Launches of several requests with enough tokens do not use the split at all: lsattn_decode_attention deals their
# tokens in equal shares to the waves, one partial per share and request.  The split below is what smaller launches get.)
FUSED_SPLIT_TOKENS = 1024
# Do not coarsen below this many (upper-bound estimate of) stage-1 workgroups: one per CU.  Measured on 131072 tokens in
# all (1 x 131072 ... 16 x 8192, 8 KV heads): 92-95 us at 256 workgroups of 1024 tokens against 100-104 us at 1024 of 256.
FUSED_MIN_WORKGROUPS = 256


# Very long contexts go further, up to 4096 tokens, while the longest request still has this many blocks: there the last,
# partly filled block of a request and the spread of lengths in the batch (which the host does not see) weigh little, and
# the partials and their merge are what is left to save (one request of 1048576 tokens: 721 -> 675 us; four of 131072
# with 32 KV heads: 1336 -> 1313 us).  With fewer blocks per request the coarser split loses to the ragged tail
# (config 3, lengths 4096..32768: 903 us at 1024, 947 at 2048).
FUSED_LONG_SPLIT_TOKENS = 4096
FUSED_LONG_MIN_BLOCKS = 64
# ... and only in batches of at most this many requests.  What the coarser split wins is a few percent and only if the
# requests are about as long as each other (64 x 65536 tokens 2.78 ms at 1024, 2.58 at 4096; 32 x 131072 2.65 at 2048,
# 2.58 at 4096); what it loses when one long request stands among many short ones is more (131072 + 255 x 512 tokens:
# 0.181 ms at 1024, 0.198 at 2048, 0.238 at 4096; 131072 + 63 x 2048: 0.207 / 0.217 / 0.275; but 524288 + 63 x 2048, where the
# long request is four fifths of all tokens: 0.447 / 0.429 / 0.416), and the larger the batch the likelier the latter.
FUSED_LONG_MAX_BATCH = 64


@functools.lru_cache(maxsize=4096)
def _fused_block_seq(block_seq: int, batch_size: int, max_len_in_batch: int, num_kv_heads: int) -> int:
    bs = int(block_seq)
    task_groups = (int(num_kv_heads) + 3) // 4
    while bs * 2 <= FUSED_LONG_SPLIT_TOKENS and bs < int(max_len_in_batch):
        blocks = (int(max_len_in_batch) + 2 * bs - 1) // (2 * bs)
        if int(batch_size) * blocks * task_groups < FUSED_MIN_WORKGROUPS:
            break
        if bs * 2 > FUSED_SPLIT_TOKENS and (blocks < FUSED_LONG_MIN_BLOCKS or int(batch_size) > FUSED_LONG_MAX_BATCH):
            break
        bs *= 2
    return bs


def longserve_token_decode_attention_flash_decoding(q, req_to_token_indexs, b_req_idx, b_seq_len, mid_o,
                                                    mid_o_logexpsum, batch_size, max_len_in_batch, q_head_num,
                                                    head_dim, cache_k, cache_v, BLOCK_SEQ, out=None,
                                                    o_logexpsum=None):
    split = _fused_block_seq(BLOCK_SEQ, batch_size, max_len_in_batch, cache_k.shape[1])
    done = _native.token_decode_attention(q, req_to_token_indexs, b_req_idx, b_seq_len, mid_o, mid_o_logexpsum, batch_size,
                                          max_len_in_batch, q_head_num, head_dim, cache_k, cache_v, split, out, o_logexpsum,
                                          longserve_cuda_kernels.FUSED_PARTIALS_BY_REQUEST)
    if done is not None:
        return done
    calcu_shape1 = (-1, q_head_num, head_dim)
    # outputs are float32 whatever q is, so that they can be merged again (FDPY:9-10)
    o_tensor = torch.empty_like(q, dtype=torch.float32) if out is None else out
    out_logexpsum = (torch.empty([batch_size, q_head_num], dtype=torch.float32, device=q.device)
                     if o_logexpsum is None else o_logexpsum)
    longserve_cuda_kernels.flash_decoding(mid_o, mid_o_logexpsum, q.view(calcu_shape1), cache_k, cache_v, req_to_token_indexs,
                                          b_req_idx, b_seq_len, max_len_in_batch, o_tensor.view(calcu_shape1), out_logexpsum,
                                          split)
    return o_tensor, out_logexpsum


# ---------------------------------------------------------------------------------------------------------------------
# Decode over a pool in 8 bits, and behind a sliding window (lsattn_pool_attention); no reference counterpart.
def pool_attention_workspace_bytes(batch_size: int, q_head_num: int, kv_head_num: int, head_dim: int, max_len_in_batch: int,
                                   window: Optional[int] = None, sinks: int = 0) -> int:
    """Bytes of device memory that the two operators below need for the partials of such a call (0: none)."""
    return int(_lib.load().lsattn_pool_attention_workspace_bytes(int(batch_size), int(q_head_num), int(kv_head_num), int(head_dim),
                                                                 int(max_len_in_batch), int(window or 0), int(sinks)))


def _pool_attention(q, table, b_req_idx, b_seq_len, max_len_in_batch, cache_k, cache_v, k_scales, v_scales, window, sinks, out, lse, workspace):
    # (a window of None is 0 to the library; one of 0 would see nothing, not even the token itself)
    if window is None or window > 0:
        done = _native.pool_attention(q, table, b_req_idx, b_seq_len, max_len_in_batch, cache_k, cache_v, k_scales, v_scales, window or 0, sinks,
                                      out, lse, workspace)
        if done is not None:
            return done
    numbers = (max_len_in_batch, window, sinks)
    if _other_ints(*numbers):
        max_len, window, sinks = (None if x is None else as_int(x) for x in numbers)
        return _pool_attention(q, table, b_req_idx, b_seq_len, max_len, cache_k, cache_v, k_scales, v_scales, window, sinks, out, lse, workspace)
    # arguments the native pass does not take: say what is wrong
    _on_current_device(((q, "q"), (table, "req_to_token_indexs"), (b_req_idx, "b_req_idx"), (b_seq_len, "b_seq_len"), (cache_k, "cache_k"),
                        (cache_v, "cache_v"), (k_scales, "k_scales"), (v_scales, "v_scales"), (out, "out"), (lse, "o_logexpsum"), (workspace, "workspace")))
    if q.dtype not in (torch.float16, torch.bfloat16) or q.dim() != 3 or not q.is_contiguous():
        raise ValueError("q must be a contiguous float16 or bfloat16 [batch, heads, head_dim] tensor")
    B, Hq, D = q.shape
    if table.dtype != torch.int32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("req_to_token_indexs must be a contiguous [max_req, max_seq] int32 tensor")
    _i32vec(b_req_idx, "b_req_idx", B)
    _i32vec(b_seq_len, "b_seq_len", B)
    if cache_k.dim() != 3 or cache_k.shape != cache_v.shape or cache_k.shape[2] != D or cache_k.dtype != cache_v.dtype:
        raise ValueError("cache_k and cache_v must be [slots, kv_heads, head_dim] for q's head_dim, of one type")
    if cache_k.stride(2) != 1 or cache_v.stride(2) != 1:
        raise ValueError("cache_k and cache_v must be contiguous in head_dim")
    if D not in (64, 128):
        raise ValueError("head_dim must be 64 or 128 (got %d)" % D)
    if cache_k.shape[1] == 0 or Hq == 0 or Hq % cache_k.shape[1]:
        raise ValueError("bad head counts: Hq=%d Hkv=%d" % (Hq, cache_k.shape[1]))
    if k_scales is not None:
        _fp8_pool(cache_k, k_scales, "cache_k", "k_scales")
        _fp8_pool(cache_v, v_scales, "cache_v", "v_scales")
    elif cache_k.dtype != q.dtype:
        raise ValueError("cache_k and cache_v must have the type of q (a pool in 8 bits: longserve_fp8_decode_attention)")
    if (window is not None and int(window) < 1) or int(sinks) < 0 or int(max_len_in_batch) < 0:
        raise ValueError("window must be >= 1 (the token itself), sinks and max_len_in_batch >= 0")
    if out is not None and (out.dtype not in (torch.float16, torch.bfloat16, torch.float32) or out.shape != q.shape or not out.is_contiguous()):
        raise ValueError("out must be a contiguous float16, bfloat16 or float32 tensor of q's shape")
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (B, Hq) or not lse.is_contiguous()):
        raise ValueError("o_logexpsum must be a contiguous float32 [batch, heads] tensor")
    if workspace is not None:
        need = pool_attention_workspace_bytes(B, Hq, cache_k.shape[1], D, max_len_in_batch, window, sinks)
        if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need:
            raise ValueError("workspace must be contiguous and hold at least %d bytes (pool_attention_workspace_bytes)" % need)
    if B == 0:
        return (torch.empty_like(q, dtype=torch.float32) if out is None else out,
                torch.empty((0, Hq), dtype=torch.float32, device=q.device) if lse is None else lse)
    raise ValueError("decode attention: arguments that no kernel takes (an empty pool?)")


def longserve_fp8_decode_attention(q: torch.Tensor, req_to_token_indexs: torch.Tensor, b_req_idx: torch.Tensor, b_seq_len: torch.Tensor,
                                   max_len_in_batch: int, cache_k: torch.Tensor, cache_v: torch.Tensor, k_scales: torch.Tensor,
                                   v_scales: torch.Tensor, window: Optional[int] = None, sinks: int = 0,
                                   out: Optional[torch.Tensor] = None, o_logexpsum: Optional[torch.Tensor] = None,
                                   workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Decode attention of one new token per request over a pool that kv_scatter_fp8 writes: (o, natural log-sum-exp).

    q [batch, q_heads, head_dim] (float16 or bfloat16, head_dim 64 or 128), cache_k / cache_v the K and V heads of the pool
    (float8_e4m3fn [slots, kv_heads, head_dim], any slot and head strides that keep rows 16-byte aligned), k_scales /
    v_scales their exponent bytes [slots, kv_heads].  out (None: float32, as longserve_token_decode_attention_flash_decoding
    returns) may be float32, float16 or bfloat16.  Products and sums are float32-exact in P and V; K and V stand for exactly what the pool holds.

    window: the token sees the last `window` positions of its context (itself among them) and the first `sinks`; None: all.
    The context of a request lies in this pool as a whole when a window is given; without one, (o, log-sum-exp) of several instances merge by
    lse_merge.  Requests without tokens get o = 0, -inf.  Entries of the table that name no slot of the pool count as positions that do not exist.
    max_len_in_batch (a bound of b_seq_len) only sizes the launch and the scratch.  workspace: the caller's scratch
    (pool_attention_workspace_bytes; else torch allocates it), one for each call that may run at the same time, graphs' replays among them."""
    if k_scales is None or v_scales is None:
        raise ValueError("k_scales and v_scales: uint8 [slots, kv_heads]")
    return _pool_attention(q, req_to_token_indexs, b_req_idx, b_seq_len, max_len_in_batch, cache_k, cache_v, k_scales, v_scales, window, sinks,
                           out, o_logexpsum, workspace)


def longserve_window_decode_attention(q: torch.Tensor, req_to_token_indexs: torch.Tensor, b_req_idx: torch.Tensor, b_seq_len: torch.Tensor,
                                      max_len_in_batch: int, cache_k: torch.Tensor, cache_v: torch.Tensor, window: int, sinks: int = 0,
                                      out: Optional[torch.Tensor] = None, o_logexpsum: Optional[torch.Tensor] = None,
                                      workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """longserve_fp8_decode_attention over the 16-bit pool (cache_k / cache_v of q's type), behind a sliding window: every token sees
    the last `window` positions of its context (itself among them) and the first `sinks`.  Positions outside cost nothing."""
    if window is None:
        raise ValueError("window must be >= 1 (without one: longserve_token_decode_attention_flash_decoding)")
    return _pool_attention(q, req_to_token_indexs, b_req_idx, b_seq_len, max_len_in_batch, cache_k, cache_v, None, None, window, sinks,
                           out, o_logexpsum, workspace)
