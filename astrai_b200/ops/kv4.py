"""The KV cache in 4 bits: storing rows, reading them back, decode attention on the codes, and copies of pages.

A key or value row of ``D`` numbers (``D`` = 32, 64, 128 or 256) is held in groups of 32.  A group has a middle ``m`` and a
step ``s`` (bf16 each) and 32 codes ``c`` of four bits, and a number reads back as ``m + s * (c - 8)``: five bits a number,
3.2 times as many tokens in the memory of a bf16 pool.  With ``lo`` and ``hi`` the group's least and greatest number,
``s = bf16((hi - lo) / 15)``, ``m = bf16(lo + 8 s)`` and ``c = clamp(round((x - m) / s), -8, 7) + 8``, so a number is off by
at most ``s / 2 + 2^-8 |m|``.  A group of equal numbers (or whose step is below 2^-120) holds its least number; a group with
an infinity or a NaN, or that spreads over 2^120 or more, reads back as NaN.

Pools: codes ``uint8 [slots, heads, D / 2]`` and ``(m, s)`` ``bf16 [slots, heads, D / 32, 2]``, the same shapes for keys and
values.  The codes of a row are held in the order in which the lanes of the attention kernel take them (``kv4.cuh``); that
order is the kernels' own affair - rows go in and out through the functions here.

On CUDA the functions run the kernels of ``kv4.cu`` (bf16 rows); the statements in plain PyTorch below are the CPU path and
the oracle of the tests.  The reference has no quantised cache.
"""

from __future__ import annotations

import functools
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from astrai_b200.ops import native

HEAD_DIMS = (32, 64, 128, 256)
GROUP = 32


@functools.lru_cache(maxsize=None)
def _op(name: str):
    return getattr(native.require(), name).default


# ------------------------------------------------------------------------------------------------ plain statements
def _check_dim(dim: int):
    if dim not in HEAD_DIMS:
        raise ValueError(f"a 4-bit cache holds rows of {', '.join(map(str, HEAD_DIMS))} numbers, not {dim}")


def pack(codes: Tensor, keys: bool) -> Tensor:
    """Codes ``[..., D]`` (0..15, in the order of the row) -> bytes ``[..., D / 2]`` in the order of the cache."""
    lead, d = codes.shape[:-1], codes.shape[-1]
    g = d // GROUP
    if keys:
        four = min(g, 4)
        codes = codes.reshape(*lead, g // four, four, 4, 8).transpose(-2, -3)
    else:
        codes = codes.reshape(*lead, g, 8, 4).transpose(-2, -3)
    codes = codes.reshape(*lead, d // 2, 2).to(torch.uint8)
    return codes[..., 0] | (codes[..., 1] << 4)


def unpack(data: Tensor, keys: bool) -> Tensor:
    """The reverse of :func:`pack`."""
    lead, d = data.shape[:-1], 2 * data.shape[-1]
    g = d // GROUP
    codes = torch.stack((data & 15, data >> 4), dim=-1)
    if keys:
        four = min(g, 4)
        return codes.reshape(*lead, g // four, 4, four, 8).transpose(-2, -3).reshape(*lead, d)
    return codes.reshape(*lead, 8, g, 4).transpose(-2, -3).reshape(*lead, d)


def quantize(x: Tensor, keys: bool) -> Tuple[Tensor, Tensor]:
    """Rows ``[..., D]`` -> codes ``uint8 [..., D / 2]`` and ``(m, s)`` ``bf16 [..., D / 32, 2]``, in plain PyTorch."""
    _check_dim(x.shape[-1])
    x = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    spread = hi - lo
    bad = ~torch.isfinite(x).all(-1, keepdim=True) | ~(spread < 2.0 ** 120)
    s = (spread / 15).to(torch.bfloat16)
    s = torch.where(bad | (s.float() < 2.0 ** -120), torch.zeros_like(s), s)
    s32 = s.float()
    m = torch.where(s32 > 0, lo + 8 * s32, lo).to(torch.bfloat16)
    m = torch.where(bad, torch.full_like(m, float("nan")), m)
    codes = torch.where(s32 > 0, ((x - m.float()) / s32).round().clamp(-8, 7) + 8, torch.full_like(x, 8.0))
    return pack(codes.to(torch.uint8).flatten(-2), keys), torch.cat((m, s), dim=-1)


def dequantize(codes: Tensor, meta: Tensor, keys: bool) -> Tensor:
    """The fp32 numbers ``[..., D]`` that codes and ``(m, s)`` stand for, in plain PyTorch."""
    c = unpack(codes, keys).float().unflatten(-1, (-1, GROUP)) - 8
    return (meta[..., :1].float() + meta[..., 1:].float() * c).flatten(-2)


def _inside(loc: Tensor, slots: int) -> Tensor:
    return (loc >= 0) & (loc < slots)


# ------------------------------------------------------------------------------------------------------ operators
def kv4_append_(k: Tensor, v: Tensor, k_codes: Tensor, k_meta: Tensor, v_codes: Tensor, v_meta: Tensor, loc: Tensor) -> None:
    """Store the rows ``k / v [tokens, heads, D]`` into the slots ``loc [tokens]`` (int32 or int64) of the pools.  A slot
    outside the pool is skipped; a slot that occurs twice ends up with a mixture of its rows, so callers name each once."""
    if k_codes.is_cuda:
        _op("kv4_append_")(k, v, k_codes, k_meta, v_codes, v_meta, loc)
        return
    if k.shape != v.shape or k.dim() != 3 or loc.shape != k.shape[:1] or k.shape[1:] != (k_codes.shape[1], 2 * k_codes.shape[2]):
        raise ValueError("kv4_append_: k / v must be [tokens, heads, head_dim] of the pools' heads and head_dim, loc [tokens]")
    ok = _inside(loc, k_codes.shape[0])
    at = loc[ok].long()
    for x, codes, meta, keys in ((k, k_codes, k_meta, True), (v, v_codes, v_meta, False)):
        codes[at], meta[at] = quantize(x[ok], keys)


def kv4_gather(k_codes: Tensor, k_meta: Tensor, v_codes: Tensor, v_meta: Tensor, loc: Tensor) -> Tuple[Tensor, Tensor]:
    """The rows of the slots ``loc [tokens]`` as bf16 ``(k, v)`` ``[tokens, heads, D]``, each number rounded once.  A slot
    outside the pool reads as zeros."""
    if k_codes.is_cuda:
        return _op("kv4_gather")(k_codes, k_meta, v_codes, v_meta, loc)
    if loc.dim() != 1:
        raise ValueError("kv4_gather: loc must be [tokens]")
    ok = _inside(loc, k_codes.shape[0])
    at = torch.where(ok, loc, torch.zeros_like(loc)).long()
    k, v = dequantize(k_codes[at], k_meta[at], True), dequantize(v_codes[at], v_meta[at], False)
    return tuple(torch.where(ok[:, None, None], x, torch.zeros_like(x)).to(torch.bfloat16) for x in (k, v))


def kv4_decode_workspace(batch: int, n_q_heads: int, n_kv_heads: int, head_dim: int, device, parts: int = 32):
    """Scratch of :func:`kv4_decode` for up to ``batch`` requests: ``(o_part, ml_part, counters)``, with room for ``parts``
    partial results per request on average (fewer than 32 can leave a part of the GPU idle when there are few requests).  Calls that may run at the
    same time (two streams, two captured graphs replayed side by side) need a workspace each."""
    return (torch.empty((batch, n_q_heads, parts, head_dim), dtype=torch.float32, device=device),
            torch.empty((batch, n_q_heads, parts, 2), dtype=torch.float32, device=device),
            torch.zeros(batch * n_kv_heads, dtype=torch.int32, device=device))


def kv4_decode(q: Tensor, k_codes: Tensor, k_meta: Tensor, v_codes: Tensor, v_meta: Tensor, req_to_token: Tensor,
               req_pool_indices: Tensor, seq_lens: Tensor, k_new: Optional[Tensor] = None, v_new: Optional[Tensor] = None, *,
               scale: Optional[float] = None, max_len: int = 0, workspace=None, out: Optional[Tensor] = None) -> Tensor:
    """Attention of one query per request over its rows of the 4-bit pools.

    ``q [batch, heads, D]``; request ``i`` has ``seq_lens[i]`` positions (int64) whose slots are
    ``req_to_token[req_pool_indices[i], :seq_lens[i]]`` (int32).  ``k_new`` / ``v_new [batch, kv_heads, D]`` are stored
    into the last position's slot first (when absent, the pool already holds them; two requests must not store into one slot).  A request of length 0 gives zeros;
    positions whose slot is outside the pool are left out.  The numbers of the cache enter unrounded, sums and softmax are
    fp32, the result is bf16.  A value's weight times its group's step is rounded to fp16 (2^-11 of it; where it is below
    2^-28 of the largest step among 32 neighbouring positions of the head, 2^-39 of that step), and query numbers below 2^-26
    of their head's largest are rounded (2^-34 of that number).

    The keys of the whole batch are spread evenly over the GPU, whatever the lengths.  ``max_len``: the longest length, when
    the host knows it (0: the table's width) - it sizes the launch, a longer request is served all the same.  ``workspace``:
    see :func:`kv4_decode_workspace`; without one the call allocates its own scratch.  On CUDA no derivative is recorded."""
    scale = float(scale) if scale is not None else q.shape[-1] ** -0.5
    if k_codes.is_cuda:
        o_part, ml_part, counters = workspace if workspace is not None else (None, None, None)
        if out is None:
            return _op("kv4_decode")(q, k_codes, k_meta, v_codes, v_meta, req_to_token, req_pool_indices, seq_lens, k_new, v_new,
                                     scale, max_len, o_part, ml_part, counters)
        _op("kv4_decode_")(q, k_codes, k_meta, v_codes, v_meta, req_to_token, req_pool_indices, seq_lens, k_new, v_new, scale,
                           max_len, o_part, ml_part, counters, out)
        return out
    hkv, slots = k_codes.shape[1], k_codes.shape[0]
    if q.dim() != 3 or req_to_token.dim() != 2 or not req_pool_indices.shape == seq_lens.shape == q.shape[:1]:
        raise ValueError("kv4_decode: q must be [batch, heads, head_dim], req_to_token [rows, positions], req_pool_indices and seq_lens [batch]")
    b, hq, d = q.shape
    if d != 2 * k_codes.shape[2] or hq % hkv:
        raise ValueError("kv4_decode: q must be [batch, heads, head_dim] with heads a multiple of the pools' heads")
    if (k_new is None) != (v_new is None):
        raise ValueError("kv4_decode: k_new and v_new come together")
    if any(t is not None and t.shape != (b, hkv, d) for t in (k_new, v_new)) or (out is not None and out.shape != q.shape):
        raise ValueError("kv4_decode: k_new / v_new must be [batch, kv_heads, head_dim] and out of q's shape")
    width, rows = req_to_token.shape[1], req_to_token.shape[0]
    res = torch.zeros_like(q, memory_format=torch.contiguous_format) if out is None else out.zero_()
    spans = []
    for row, n in zip(req_pool_indices.tolist(), seq_lens.tolist()):
        n = min(max(n, 0), width) if 0 <= row < rows else 0
        spans.append(req_to_token[row, :n].long() if n else req_to_token.new_zeros(0).long())
    if k_new is not None:
        last = torch.tensor([int(s[-1]) if s.numel() else -1 for s in spans], dtype=torch.long)
        kv4_append_(k_new, v_new, k_codes, k_meta, v_codes, v_meta, last)
    for i, span in enumerate(spans):
        span = span[_inside(span, slots)]
        if not span.numel():
            continue
        k, v = dequantize(k_codes[span], k_meta[span], True), dequantize(v_codes[span], v_meta[span], False)
        p = torch.einsum("hgd,lhd->hgl", q[i].float().view(hkv, hq // hkv, d), k).mul(scale).softmax(-1)
        res[i] = torch.einsum("hgl,lhd->hgd", p, v).reshape(hq, d).to(res.dtype)
    return res


def copy_pages_(pools: Sequence[Tensor], src: Sequence[int], dst: Sequence[int], page_size: int) -> None:
    """Make page ``dst[i]`` of every layer of every pool a copy of page ``src[i]``: one launch for up to 256 pages.

    ``pools``: up to eight contiguous tensors ``[layers, slots, ...]`` of any type with as many layers and slots each; page
    ``p`` is the slots ``[p * page_size, (p + 1) * page_size)``.  The page numbers are host integers, checked before anything
    is written: no destination may be a source or occur twice (a source may serve several destinations)."""
    pools = list(pools)
    if pools and pools[0].is_cuda:
        _op("copy_pages_")(pools, list(src), list(dst), page_size)
        return
    src, dst = [int(p) for p in src], [int(p) for p in dst]
    if not 1 <= len(pools) <= 8:
        raise ValueError("copy_pages_: 1 to 8 pools")
    if page_size < 1 or len(src) != len(dst):
        raise ValueError("copy_pages_: page_size >= 1, as many sources as destinations")
    if any(t.shape[:2] != pools[0].shape[:2] or not t.is_contiguous() for t in pools):
        raise RuntimeError("copy_pages_: the pools must be contiguous [layers, slots, ...] tensors with as many layers and slots each")
    pages = pools[0].shape[1] // page_size
    for p in (*src, *dst):
        if not 0 <= p < pages:
            raise ValueError(f"copy_pages_: page {p} is outside the pool of {pages} pages")
    if len(set(dst)) != len(dst) or not set(dst).isdisjoint(src):
        raise ValueError("copy_pages_: a page is written twice, or both read and written")
    for t in pools:
        paged = t[:, :pages * page_size].unflatten(1, (pages, page_size))
        paged[:, dst] = paged[:, src]
