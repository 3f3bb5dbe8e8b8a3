"""Attention with a KV cache: append this step's K/V to the pool, then attend over the cached prefix + new tokens.

Packed layout: ``q [T, Hq, D]``, ``k / v [T, Hkv, D]`` where the batch is concatenated along ``T``.
* ``fwd="decode"`` (one new token per request): the split-KV paged kernel (``paged_attention.cu``) on CUDA, which also
  stores the step's K / V rows into the pool (no separate append launch);
* ``fwd="prefill"`` (ragged, possibly with a cached prefix): ONE varlen launch of the tcgen05 flash kernel
  (``flash_fwd.cu``, lower-right aligned causal mask) serves every request.  With pages of 8 / 16 / 32 / 64 tokens the
  kernel reads K / V straight from the pool through the slot table; other page sizes (and the contiguous layout's
  page size 1) gather the batch's keys into packed tensors first.  Head dims other than 64 / 128 and explicit masks
  take a per-request SDPA loop.
* a 4-bit cache (:mod:`astrai_b200.ops.kv4`): decode attends on the codes, and so does a prefill that has one position of
  each request (forks, prompts found whole in the prefix index); any other prefill stores the new rows, reads the batch's
  rows back as bf16, those of a bounded number of keys at a time, and runs the same varlen launch.
The CPU statement of both is the same gather + softmax and is what the tests compare against
(semantics of ``TorchNativeBackend`` in the reference, ``astrai/extension/backend/attention.py:443-498``).
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor

from astrai_b200.ops import flash, kv4, native
from astrai_b200.ops.kv import KVCache


def _append(k: Tensor, v: Tensor, cache: KVCache, layer_id: int):
    kb, vb = cache.k_buffer[layer_id], cache.v_buffer[layer_id]
    loc = cache.out_cache_loc.reshape(-1)
    if k.is_cuda and k.dtype == torch.bfloat16 and kb.dtype == torch.bfloat16 and (kb.shape[1] * kb.shape[2]) % 8 == 0:
        native.require()
        torch.ops.astrai_b200.kv_append_(k.contiguous(), v.contiguous(), kb, vb, loc.to(torch.int32))
    else:
        idx = loc.long()
        kb[idx] = k.to(kb.dtype)
        vb[idx] = v.to(vb.dtype)


def _gather_kv(cache: KVCache, layer_id: int, row: int, length: int):
    slots = cache.req_to_token[row, :length].long()
    if cache.four_bit:
        return kv4.kv4_gather(*cache.layer_pools(layer_id), slots)
    return cache.k_buffer[layer_id][slots], cache.v_buffer[layer_id][slots]


def _sdpa_one(q: Tensor, k: Tensor, v: Tensor, causal: bool, mask_row: Optional[Tensor] = None) -> Tensor:
    """q [S,Hq,D], k/v [L,Hkv,D]; causal is lower-right aligned (query i sees keys <= L-S+i)."""
    s, l = q.shape[0], k.shape[0]
    hq, hkv = q.shape[1], k.shape[1]
    qt, kt, vt = q.transpose(0, 1)[None], k.transpose(0, 1)[None], v.transpose(0, 1)[None]
    attn_mask = None
    if causal and not (s == l):
        i = torch.arange(s, device=q.device)[:, None]
        j = torch.arange(l, device=q.device)[None, :]
        attn_mask = j <= (l - s + i)
    if mask_row is not None:
        attn_mask = mask_row if attn_mask is None else (attn_mask & mask_row)
    if not q.is_cuda and hq != hkv:
        kt = kt.repeat_interleave(hq // hkv, dim=1)
        vt = vt.repeat_interleave(hq // hkv, dim=1)
        out = F.scaled_dot_product_attention(qt, kt, vt, attn_mask=attn_mask, is_causal=causal and attn_mask is None)
    else:
        out = F.scaled_dot_product_attention(qt, kt, vt, attn_mask=attn_mask, is_causal=causal and attn_mask is None,
                                             enable_gqa=hq != hkv)
    return out[0].transpose(0, 1)


def _lens(cache: KVCache):
    kv = cache.kv_lens if cache.kv_lens is not None else cache.seq_lens.tolist()
    if cache.q_lens is not None:
        return cache.q_lens, kv
    if cache.qo_indptr is not None:
        ptr = cache.qo_indptr.tolist()
        return [b - a for a, b in zip(ptr[:-1], ptr[1:])], kv
    return [1] * len(kv), kv


def _decode_native_ok(q: Tensor, cache: KVCache) -> bool:
    return (
        q.is_cuda and q.dtype == torch.bfloat16 and (cache.four_bit or cache.k_buffer.dtype == torch.bfloat16)
        and q.shape[-1] in (32, 64, 128, 256) and cache.decode_o_part is not None and cache.decode_counters is not None
        and q.shape[1] % cache.k_buffer.shape[2] == 0 and 1 <= q.shape[1] // cache.k_buffer.shape[2] <= 8
    )


# Bytes of bf16 rows that a prefill over a 4-bit pool reads back at a time (a longer request's rows are read at once).  A
# piece of few requests leaves the attention kernel few items: 16 requests of 64 positions behind 16320 (1 GB of rows, 32 / 8
# heads of 128) take 0.80 ms in one piece, 0.83 in two, 1.07 in three and 1.73 in six; 8 of 128 behind 65408 (2 GB) 1.58 ms in one, 2.31 in
# two, 4.13 in four.  Without a bound a batch behind long histories takes as much memory as a bf16 pool would.
READ_BACK_BYTES = 1 << 30


def read_back_pieces(kv_lens: Sequence[int], limit: int) -> List[Tuple[int, int]]:
    """Ranges ``[first, last)`` of requests, about equal, that have at most ``limit`` keys together; a longer request has its own."""
    total = sum(kv_lens)
    share = total / max(1, -(-total // max(limit, 1)))
    pieces, first, keys = [], 0, 0
    for i, n in enumerate(kv_lens):
        if i > first and (keys + n > limit or keys >= share):
            pieces.append((first, i))
            first, keys = i, 0
        keys += n
    return pieces + [(first, len(kv_lens))]


def _read_back_attention(q: Tensor, pools, cache: KVCache, q_lens, kv_lens, scale: float) -> Tensor:
    """Ragged prefill over a 4-bit pool.  The prompt's own rows are read back with the cached ones, so that the positions of a
    chunk see the same numbers of a key wherever the prompt was cut."""
    limit = READ_BACK_BYTES // (4 * pools[0].shape[1] * q.shape[-1])
    if sum(kv_lens) <= limit or len(kv_lens) == 1:
        return flash.flash_attention_ragged(q, *kv4.kv4_gather(*pools, cache.kv_gather_loc), cache.qo_indptr, cache.kv_indptr,
                                            max(q_lens), max(kv_lens), scale, rows_alone=True)
    outs, q0, k0 = [], 0, 0
    for a, b in read_back_pieces(kv_lens, limit):
        q1, k1 = q0 + sum(q_lens[a:b]), k0 + sum(kv_lens[a:b])
        outs.append(flash.flash_attention_ragged(q[q0:q1], *kv4.kv4_gather(*pools, cache.kv_gather_loc[k0:k1]), cache.qo_indptr[a:b + 1] - q0,
                                                 cache.kv_indptr[a:b + 1] - k0, max(q_lens[a:b]), max(kv_lens[a:b]), scale, rows_alone=True))
        q0, k0 = q1, k1
    return torch.cat(outs)


def _one_position_each(q: Tensor, cache: KVCache, q_lens) -> bool:
    """A prefill of at most one query of each request that the decode kernel answers: one of each, no derivative asked for.  Heads of 128, 8 forks of
    4096 positions (16 / 4 heads): 40 us, and 90 us with the rows read back; 64 of 16384 (32 / 8): 0.32 and 4.9 ms."""
    hkv = cache.k_buffer.shape[2]
    return (len(q_lens) == q.shape[0] and q.shape[1] % hkv == 0 and 1 <= q.shape[1] // hkv <= 8
            and cache.seq_lens.dtype == torch.int64 and cache.req_pool_indices.dtype == torch.int32
            and not flash.derivatives_asked(q))


def cached_attention(q: Tensor, k: Tensor, v: Tensor, kv_cache: KVCache, layer_id: int = 0,
                     attn_mask: Optional[Tensor] = None, is_causal: bool = True, fwd: str = "prefill") -> Tensor:
    if kv_cache is None:
        raise ValueError("inference attention requires a KV cache")
    if q.dim() != 3:
        raise ValueError("packed inference tensors must be [tokens, heads, head_dim]")
    scale = q.shape[-1] ** -0.5
    from astrai_b200.ops import backend as _backend

    native_on = _backend.get_backend(q.device.type) is _backend.ATTN_BACKEND.TCGEN05
    if native_on and fwd == "decode" and attn_mask is None and _decode_native_ok(q, kv_cache):
        # one launch: the step's K / V rows are stored into the pool by the attention kernel itself (the reference fuses
        # its append the same way, csrc/kernels/attention/layout_policies.cuh:221-254)
        b = q.shape[0]
        if kv_cache.four_bit:
            out = kv_cache.decode_out[:b] if kv_cache.decode_out is not None else None
            return kv4.kv4_decode(q, *kv_cache.layer_pools(layer_id), kv_cache.req_to_token, kv_cache.req_pool_indices,
                                  kv_cache.seq_lens, k_new=k, v_new=v, scale=scale, max_len=kv_cache.max_len, out=out,
                                  workspace=(kv_cache.decode_o_part, kv_cache.decode_ml_part, kv_cache.decode_counters))
        splits = kv_cache.decode_splits or int(torch.ops.astrai_b200.paged_decode_splits(
            b, kv_cache.k_buffer.shape[2], max(kv_cache.max_len, 1), kv_cache.decode_o_part.shape[2]))
        out = kv_cache.decode_out[:b] if kv_cache.decode_out is not None else torch.empty_like(q)
        torch.ops.astrai_b200.paged_decode_append_(
            q.contiguous(), k.contiguous(), v.contiguous(), kv_cache.k_buffer[layer_id], kv_cache.v_buffer[layer_id],
            kv_cache.req_to_token, kv_cache.req_pool_indices, kv_cache.seq_lens, scale, splits, kv_cache.decode_o_part,
            kv_cache.decode_ml_part, kv_cache.decode_counters, out)
        return out
    pools = kv_cache.layer_pools(layer_id) if kv_cache.four_bit else None
    if pools is not None:
        kv4.kv4_append_(k, v, *pools, kv_cache.out_cache_loc.reshape(-1))
    else:
        _append(k, v, kv_cache, layer_id)
    q_lens, kv_lens = _lens(kv_cache)
    page = getattr(kv_cache, "page_size", 1) or 1
    if pools is not None:
        if native_on and attn_mask is None and fwd == "prefill" and q.is_cuda and q.dtype == torch.bfloat16:
            if max(q_lens) == 1 and _one_position_each(q, kv_cache, q_lens):
                return kv4.kv4_decode(q, *pools, kv_cache.req_to_token, kv_cache.req_pool_indices, kv_cache.seq_lens, scale=scale,
                                      max_len=max(kv_lens))
            if kv_cache.kv_gather_loc is not None and kv_cache.qo_indptr is not None and q.shape[-1] in flash.SUPPORTED_HEAD_DIMS:
                return _read_back_attention(q, pools, kv_cache, q_lens, kv_lens, scale)
    elif (native_on and attn_mask is None and fwd == "prefill" and kv_cache.qo_indptr is not None and page in flash.PAGED_PAGE_SIZES
            and flash.supported(q, kv_cache.k_buffer[layer_id], kv_cache.v_buffer[layer_id])):
        # ragged prefill over the paged pool: the kernel walks the slot table itself (no gathered copy of the keys)
        return flash.flash_attention_paged(q, kv_cache.k_buffer[layer_id], kv_cache.v_buffer[layer_id], kv_cache.qo_indptr,
                                           kv_cache.kv_indptr, kv_cache.req_to_token, kv_cache.req_pool_indices, page,
                                           max(q_lens), causal=True, scale=scale)
    if (not kv_cache.four_bit and native_on and attn_mask is None and fwd == "prefill" and kv_cache.kv_gather_loc is not None
            and kv_cache.qo_indptr is not None and flash.supported(q, kv_cache.k_buffer[layer_id], kv_cache.v_buffer[layer_id])):
        # ragged prefill on the tcgen05 flash kernel: gather this batch's keys / values from the pool (cached prefix
        # included) into packed tensors once, then one varlen launch with lower-right aligned causal masking
        kk = kv_cache.k_buffer[layer_id].index_select(0, kv_cache.kv_gather_loc)
        vv = kv_cache.v_buffer[layer_id].index_select(0, kv_cache.kv_gather_loc)
        return flash.flash_attention_ragged(q, kk, vv, kv_cache.qo_indptr, kv_cache.kv_indptr, max(q_lens), max(kv_lens), scale)
    rows = kv_cache.req_pool_indices.tolist()
    outs, start = [], 0
    for i, (ql, kl) in enumerate(zip(q_lens, kv_lens)):
        kk, vv = _gather_kv(kv_cache, layer_id, rows[i], kl)
        mask_row = None
        if attn_mask is not None:
            mask_row = attn_mask[i].reshape(-1, attn_mask.shape[-1])[..., :kl].bool()
        causal = is_causal or fwd == "decode" or ql > 1
        outs.append(_sdpa_one(q[start:start + ql], kk.to(q.dtype), vv.to(q.dtype), causal and ql > 1, mask_row))
        start += ql
    return torch.cat(outs, dim=0)
