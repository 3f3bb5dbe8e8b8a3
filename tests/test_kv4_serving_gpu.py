"""Serving over a 4-bit KV cache on the GPU: prefill behind long cached histories, forks, captured decode steps."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rows(*shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * torch.exp(torch.randn(shape[-1], device="cuda", generator=g) * 0.5)).bfloat16()


def _cached(lens, heads, kv_heads, dim, page=16):
    """A pool whose slots all hold rows, a manager with a task of each length, their workspace."""
    from astrai_b200 import ops
    from astrai_b200.inference.cache import PagePool, TaskCacheManager
    from astrai_b200.inference.workspace import InferenceWorkspace

    longest, b = max(lens), len(lens)
    tokens = sum(-(-n // page) for n in lens) * page
    pool = PagePool(1, kv_heads, dim, b, longest, "cuda", torch.bfloat16, page_size=page, n_tokens=tokens, kv_dtype="int4")
    tc = TaskCacheManager(pool)
    ws = InferenceWorkspace(b, longest, heads, dim, "cuda", torch.bfloat16, n_kv_heads=kv_heads, max_prefill_tokens=1024)
    for i, n in enumerate(lens):
        assert tc.task_alloc(f"t{i}", [i * 100000 + j for j in range(n)])
    st = pool.storage
    for at in torch.arange(tokens, device="cuda").split(16384):
        ops.kv4_append_(_rows(len(at), kv_heads, dim, seed=int(at[0])), _rows(len(at), kv_heads, dim, seed=int(at[0]) + 1),
                        *(t[0] for t in (st.k_buffer, st.k_meta, st.v_buffer, st.v_meta)), at)
    return pool, tc, ws


def _expected(pool, kv, q, counts, kv_lens, i, scale):
    """64-bit attention of request ``i`` over what its cache holds, ``[queries, heads, D]``, and how far a result may be off.

    Rows are read back as bf16 (2^-8 of each number) and the probabilities enter the second product as bf16 (2^-8): the sum
    is off by 2 x 2^-8 sum p |v| from those; a logit is off by 2^-8 scale sum |q k| =: d at most, which changes p by 2 d p
    and, through the sum of the softmax, the result by as much again; the result's rounding is 2^-8 |o|.  The decode kernel
    takes the rows unrounded and multiplies codes (0..15) by ``p s`` in fp16 instead: 2^-11 sum p s 15."""
    from astrai_b200.ops import kv4

    start, n, c = sum(counts[:i]), kv_lens[i], counts[i]
    st, slots = pool.storage, kv.req_to_token[int(kv.req_pool_indices[i]), :n].long()
    k, v = (kv4.dequantize(b[0][slots], m[0][slots], keys).double().repeat_interleave(q.shape[1] // b.shape[2], 1) for b, m, keys in
            ((st.k_buffer, st.k_meta, True), (st.v_buffer, st.v_meta, False)))
    qd = q[start:start + c].double()
    seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - c, n, device="cuda")[:, None]
    p = torch.softmax((torch.einsum("shd,lhd->hsl", qd, k) * scale).masked_fill(~seen, -math.inf), -1)
    d = torch.einsum("shd,lhd->hsl", qd.abs(), k.abs()) * scale * 2.0 ** -8
    o, size = torch.einsum("hsl,lhd->shd", p, v), torch.einsum("hsl,lhd->shd", p, v.abs())
    coded = torch.einsum("hsl,lhd->shd", p, st.v_meta[0][slots][..., 1].double().repeat_interleave(32, -1).repeat_interleave(q.shape[1] // pool.n_kv_heads, 1) * 15)
    moved = 2 * torch.einsum("hsl,lhd->shd", p * d, v.abs()) + 2 * size * (p * d).sum(-1).t()[..., None]
    return o, 2.0 ** -8 * o.abs() + 2 * 2.0 ** -8 * size + 2.0 ** -11 * coded + moved


def _attend(pool, tc, ws, counts, lens, heads, kv_heads, dim):
    """``ops.attention`` of the last ``counts`` positions of each request; the result, the cache and the memory it took."""
    from astrai_b200 import ops

    kv = tc.bind([f"t{i}" for i in range(len(lens))], ws, start_positions=[n - c for n, c in zip(lens, counts)])
    q, k, v = (_rows(sum(counts), h, dim, seed=70 + j) for j, h in enumerate((heads, kv_heads, kv_heads)))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = ops.attention(q, k, v, kv, 0, None, True, "prefill")
    torch.cuda.synchronize()
    return q, kv, out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 8, 128), (4, 4, 64), (4, 2, 256), (2, 2, 32)])
def test_forks_of_a_long_prompt_read_nothing_back(heads, kv_heads, dim):
    """One position of each request (a fork, a prompt found whole in the prefix index): attention on the codes."""
    lens = [4001 + 3 * i for i in range(24)]
    pool, tc, ws = _cached(lens, heads, kv_heads, dim)
    counts = [1] * len(lens)
    q, kv, out, taken = _attend(pool, tc, ws, counts, lens, heads, kv_heads, dim)
    assert taken < 16 << 20, f"{taken >> 20} MB of scratch"  # the rows themselves would be 24 x 4036 x kv_heads x dim x 4 bytes
    for i in (0, 11, 23):
        o, tol = _expected(pool, kv, q, counts, lens, i, dim ** -0.5)
        assert ((out[i:i + 1].double() - o).abs() <= tol).all()


def test_a_batch_reads_its_histories_back_in_bounded_pieces(monkeypatch):
    """Few new positions behind long histories: the rows of a bounded number of keys are there at a time."""
    from astrai_b200.ops import paged_attention

    heads, kv_heads, dim = 4, 2, 128
    lens, counts = [3000, 40, 2999, 7, 3003, 2500, 9000, 64], [5, 1, 1, 7, 130, 2, 3, 64]
    pool, tc, ws = _cached(lens, heads, kv_heads, dim)
    whole = _attend(pool, tc, ws, counts, lens, heads, kv_heads, dim)[2]
    limit = 4 * 4000 * kv_heads * dim
    monkeypatch.setattr(paged_attention, "READ_BACK_BYTES", limit, raising=False)
    q, kv, out, taken = _attend(pool, tc, ws, counts, lens, heads, kv_heads, dim)
    # the longest request alone (9000 keys), and small change for offsets and results
    assert taken < 4 * 9000 * kv_heads * dim + (2 << 20), f"{taken} bytes of scratch"
    assert torch.equal(out, whole)  # a request's sums do not depend on the others
    for i in range(len(lens)):
        o, tol = _expected(pool, kv, q, counts, lens, i, dim ** -0.5)
        assert ((out[sum(counts[:i]):sum(counts[:i + 1])].double() - o).abs() <= tol).all()


def test_a_table_whose_positions_would_pass_32_bits_is_refused():
    """Positions are counted in 32 bits, some turns beyond a request's last one; the table itself is never read here."""
    from astrai_b200 import ops

    pools = [t for _ in "kv" for t in (torch.zeros(16, 1, 32, dtype=torch.uint8, device="cuda"), torch.zeros(16, 1, 2, 2, dtype=torch.bfloat16, device="cuda"))]
    q, rows = _rows(1, 1, 64, seed=1), torch.zeros(1, dtype=torch.int32, device="cuda")
    table = torch.empty(1, 2 ** 31 - 512, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="table too large"):
        ops.kv4_decode(q, *pools, table, rows, torch.zeros(1, dtype=torch.int64, device="cuda"))
