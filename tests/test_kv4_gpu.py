"""The kernels of the 4-bit KV cache against plain statements in 64 bits (``kv4.cu``)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DIMS = (32, 64, 128, 256)


def _pools(slots, heads, dim, layers=None):
    lead = (slots, heads) if layers is None else (layers, slots, heads)
    return [t for _ in "kv" for t in (torch.zeros(*lead, dim // 2, dtype=torch.uint8, device="cuda"),
                                      torch.zeros(*lead, dim // 32, 2, dtype=torch.bfloat16, device="cuda"))]


def _rows(*shape, seed, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = torch.exp(torch.randn(shape[-1], device="cuda", generator=g) * 0.7)
    return (torch.randn(*shape, device="cuda", generator=g) * wide + offset * torch.randn(shape[-1], device="cuda", generator=g)).bfloat16()


def _same_meta(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=-7e30), torch.nan_to_num(b.float(), nan=-7e30))


# ------------------------------------------------------------------------------------------------------ rows in and out
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("tokens,heads,loc_dtype", [(1, 1, torch.int32), (37, 3, torch.int64), (300, 4, torch.int32), (5, 8, torch.int64)])
def test_rows_in_and_out_are_exact(tokens, heads, dim, loc_dtype):
    """Codes, middles and steps come from IEEE single arithmetic, so they are the plain statement's bit for bit; a number
    read back is ``m + s (c - 8)`` (the product has 12 bits) rounded once to fp32 and once to bf16, as in the statement."""
    from astrai_b200 import ops
    from astrai_b200.ops import kv4

    slots = 2 * tokens + 5
    k, v = _rows(tokens, heads, dim, seed=1), _rows(tokens, heads, dim, seed=2)
    if tokens > 4:
        k[0], k[1, 0, 3], v[2, -1, 0] = 1.25, math.inf, math.nan
        v[3, 0, :2] = torch.tensor([2.0 ** 119, -2.0 ** 119])
        k[4, 0, 1] = 2.0 ** -130  # subnormal
        v[4] = v[4] * 1e-38
    loc = torch.randperm(slots, device="cuda")[:tokens].to(loc_dtype)
    pools = _pools(slots, heads, dim)
    for t in pools:
        t.fill_(77)
    before = [t.clone() for t in pools]
    ops.kv4_append_(k, v, *pools, loc)
    at = loc.long()
    others = torch.ones(slots, dtype=torch.bool, device="cuda")
    others[at] = False
    for i, (x, keys) in enumerate(((k, True), (v, False))):
        codes, meta = kv4.quantize(x.cpu(), keys)
        assert torch.equal(pools[2 * i][at].cpu(), codes) and _same_meta(pools[2 * i + 1][at].cpu(), meta)
    assert all(torch.equal(t[others], b[others]) for t, b in zip(pools, before))  # the other slots are left as they were
    got = ops.kv4_gather(*pools, loc)
    for i, keys in enumerate((True, False)):
        want = kv4.dequantize(pools[2 * i][at].cpu(), pools[2 * i + 1][at].cpu(), keys).bfloat16()
        assert _same_meta(got[i].cpu(), want)


def test_slots_outside_the_pool_and_strided_rows():
    from astrai_b200 import ops
    from astrai_b200.ops import kv4

    qkv = _rows(6, 12, 64, seed=3)
    k, v = qkv[:, 4:8], qkv[:, 8:]  # views of a fused projection
    odd = _rows(6, 4, 65, seed=4)[..., :64]  # rows that do not start on 16 bytes
    for kk, vv in ((k, v), (odd, v)):
        pools = _pools(9, 4, 64)
        loc = torch.tensor([8, -1, 0, 9, 2 ** 40, 3], device="cuda")
        ops.kv4_append_(kk, vv, *pools, loc)
        assert not pools[0][[1, 2, 4, 5, 6, 7]].any()
        gk, gv = ops.kv4_gather(*pools, loc)
        for got, x, keys in ((gk, kk, True), (gv, vv, False)):
            want = kv4.dequantize(*kv4.quantize(x.cpu(), keys), keys).bfloat16()
            want[[1, 3, 4]] = 0
            assert torch.equal(got.cpu(), want)


def test_contiguous_rows_and_queries_that_start_off_a_16_byte_boundary():
    from astrai_b200 import ops

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        return flat[1:].view(t.shape).copy_(t)

    k, v, q = _rows(5, 2, 64, seed=5), _rows(5, 2, 64, seed=6), _rows(1, 4, 64, seed=7)
    loc = torch.arange(5, device="cuda")
    table, row, lens = torch.arange(5, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([5], device="cuda")
    results = []
    for put in (lambda t: t, shifted):
        pools = _pools(6, 2, 64)
        ops.kv4_append_(put(k), put(v), *pools, loc)
        out = ops.kv4_decode(put(q), *pools, table, row, lens, k_new=put(k[:1].clone()), v_new=put(v[:1].clone()), max_len=5)
        results.append((*pools, out))
    assert all(torch.equal(a, b) for a, b in zip(*results))


# ---------------------------------------------------------------------------------------------------------- attention
def _case(lens, heads, kv_heads, dim, seed, page=4, spare=3):
    """Pools whose slots outside the requests' positions read as NaN, a table, queries and a step's rows."""
    from astrai_b200 import ops

    g = torch.Generator().manual_seed(seed)
    width = max(max(lens), 1)
    per = [-(-n // page) for n in lens]
    pages = torch.randperm(sum(per) + spare, generator=g)
    table = torch.full((len(lens) + 2, width), -5, dtype=torch.int32)
    order = torch.randperm(len(lens) + 2, generator=g)[:len(lens)]
    start = 0
    for i, (n, p) in enumerate(zip(lens, per)):
        slots = (pages[start:start + p, None] * page + torch.arange(page)).reshape(-1)[:n]
        table[order[i], :n] = slots.int()
        start += p
    slots = len(pages) * page
    pools = _pools(slots, kv_heads, dim)
    for t in (pools[1], pools[3]):
        t.fill_(math.nan)
    used = torch.cat([table[order[i], :n] for i, n in enumerate(lens)]).long().cuda()
    n = used.numel()
    ops.kv4_append_(_rows(n, kv_heads, dim, seed=seed + 1), _rows(n, kv_heads, dim, seed=seed + 2, offset=0.2), *pools, used)
    gd = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(len(lens), heads, dim, device="cuda", generator=gd).bfloat16()
    new = (_rows(len(lens), kv_heads, dim, seed=seed + 3), _rows(len(lens), kv_heads, dim, seed=seed + 4))
    return pools, table.cuda(), order.int().cuda(), torch.tensor(lens, device="cuda"), q, new


def _expected(pools, table, rows, lens, q, scale):
    """64-bit attention and, number by number, how far the kernel's result may be off.

    The result's rounding to bf16: 2^-8 |o|.  The kernel multiplies the values' codes (0..15, whole numbers) by
    ``p s`` in fp16: off by at most 2^-11 p s 15 a key.  Logits are sums in fp32 of products that are at most
    |q| (|m| + 15 s); with fewer than 2^9 roundings of 2^-23 each they are off by ``d = 2^-14`` times the mean size of
    a partial sum over the products - taken as 2^-18 of the sum of all their sizes - and a softmax whose logits are off
    by d changes p by a factor of at most 1 + 2d (+ 2^-21 for the exponential)."""
    from astrai_b200.ops import kv4

    outs, tols = [], []
    slots_n, (hq, dim), hkv = pools[0].shape[0], q.shape[1:], pools[0].shape[1]
    for i, n in enumerate(lens.tolist()):
        n = min(n, table.shape[1])
        row = int(rows[i])
        slots = table[row, :n].long() if 0 <= row < table.shape[0] else table[0, :0].long()
        slots = slots[(slots >= 0) & (slots < slots_n)]
        if not slots.numel():
            outs.append(torch.zeros(hq, dim, dtype=torch.double, device="cuda"))
            tols.append(torch.zeros(hq, dim, dtype=torch.double, device="cuda"))
            continue
        k, v = (kv4.dequantize(pools[j][slots], pools[j + 1][slots], j == 0).double().repeat_interleave(hq // hkv, 1) for j in (0, 2))
        ms, ss = (pools[j][slots].double().repeat_interleave(32, -2).repeat_interleave(hq // hkv, 1) for j in (1, 3))
        qd = q[i].double()
        p = torch.softmax(torch.einsum("hd,lhd->hl", qd, k) * scale, -1)
        o = torch.einsum("hl,lhd->hd", p, v)
        size = torch.einsum("hd,lhd->hl", qd.abs(), ms[..., 0].abs() + 15 * ms[..., 1]).amax(-1) * scale
        d = 2.0 ** -18 * size + 2.0 ** -21
        coded = torch.einsum("hl,lhd->hd", p, ss[..., 1] * 15)
        spread = torch.einsum("hl,lhd->hd", p, v.abs())
        outs.append(o)
        tols.append(2.0 ** -8 * o.abs() + 2.0 ** -11 * coded + 2 * d[:, None] * spread + 1e-30)
    return torch.stack(outs), torch.stack(tols)


def _near(out, want):
    o, tol = want
    off = (out.double() - o).abs()
    assert torch.isfinite(out).all()
    assert (off <= tol).all(), f"off by {(off / tol.clamp(min=1e-30)).max().item():.2f} of the tolerance"


LENS = [[1], [1, 0, 33, 32, 31], [130, 2, 257, 64], [700, 1, 5], [0, 0]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (6, 2), (8, 1), (15, 3), (28, 4)])
@pytest.mark.parametrize("dim", DIMS)
def test_decode_attention(lens, heads, kv_heads, dim):
    from astrai_b200 import ops

    pools, table, rows, n, q, new = _case(lens, heads, kv_heads, dim, seed=heads + dim)
    scale = dim ** -0.5
    for parts in (None, 2, 3, 32):  # two parts: a single CTA walks every request
        work = parts and ops.kv4_decode_workspace(len(lens), heads, kv_heads, dim, "cuda", parts=parts)
        _near(ops.kv4_decode(q, *pools, table, rows, n, workspace=work), _expected(pools, table, rows, n, q, scale))
    # with the step's own rows: stored first, then attended to
    stored = [t.clone() for t in pools]
    live = n > 0
    last = table[rows.long(), (n - 1).clamp(min=0)]
    ops.kv4_append_(new[0][live], new[1][live], *stored, last[live])
    out = ops.kv4_decode(q, *pools, table, rows, n, *new, scale=0.31, max_len=max(lens), workspace=ops.kv4_decode_workspace(len(lens), heads, kv_heads, dim, "cuda"))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pools, stored))
    _near(out, _expected(pools, table, rows, n, q, 0.31))


@pytest.mark.parametrize("page", [1, 16])
def test_long_and_many_requests(page):
    from astrai_b200 import ops

    for lens, heads, kv_heads, dim in (([9001], 8, 2, 128), ([300 + 7 * i for i in range(70)], 4, 1, 64)):
        pools, table, rows, n, q, _ = _case(lens, heads, kv_heads, dim, seed=5, page=page)
        _near(ops.kv4_decode(q, *pools, table, rows, n), _expected(pools, table, rows, n, q, dim ** -0.5))


def test_more_requests_than_threads_a_short_max_len_and_many_heads():
    from astrai_b200 import ops

    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 90, (300,), generator=g).tolist()  # a thread finds the place of several requests
    lens[150] = 1500
    for lens, heads, kv_heads, dim in ((lens, 2, 1, 64), ([500, 3, 0, 129], 128, 64, 32), ([40, 2], 512, 512, 32)):
        pools, table, rows, n, q, _ = _case(lens, heads, kv_heads, dim, seed=31)
        want = _expected(pools, table, rows, n, q, dim ** -0.5)
        for parts, max_len in ((2, 0), (3, 7), (32, 1), (32, 0)):  # lengths beyond max_len are served all the same
            work = ops.kv4_decode_workspace(len(lens) + 3, heads, kv_heads, dim, "cuda", parts=parts)  # and the workspace may be larger
            _near(ops.kv4_decode(q, *pools, table, rows, n, max_len=max_len, workspace=work), want)
            assert not work[2].any()


def test_no_rows_views_of_a_projection_and_a_request_named_twice():
    from astrai_b200 import ops

    pools, table, rows, n, _, _ = _case([50, 9, 33], 4, 2, 64, seed=33)
    before = [t.clone() for t in pools]
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    ops.kv4_append_(none, none, *pools, torch.empty(0, dtype=torch.int32, device="cuda"))
    got = ops.kv4_gather(*pools, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert [t.shape for t in got] == [(0, 2, 64)] * 2
    qkv = _rows(3, 8, 64, seed=34)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    out = ops.kv4_decode(q, *pools, table, rows, n, k, v)
    pools2 = [t.clone() for t in before]
    assert torch.equal(out, ops.kv4_decode(q.contiguous(), *pools2, table, rows, n, k.contiguous(), v.contiguous()))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pools, pools2))
    twice = rows[[0, 0, 2]]
    _near(ops.kv4_decode(q, *pools, table, twice, n[[0, 0, 2]]), _expected(pools, table, twice, n[[0, 0, 2]], q, 64 ** -0.5))


def test_a_graph_serves_lengths_that_grow_and_two_streams_run_side_by_side():
    from astrai_b200 import ops

    pools, table, rows, n, q, new = _case([900, 300, 0, 777], 8, 2, 128, seed=35)
    full = n.clone()
    n.copy_((full > 0).long())
    work, out, g = ops.kv4_decode_workspace(4, 8, 2, 128, "cuda"), torch.empty_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv4_decode(q, *pools, table, rows, n, *new, workspace=work, out=out)
    for part in (0.0, 0.3, 1.0):
        n.copy_(torch.maximum((full * part).long(), (full > 0).long()))
        g.replay()
        _near(out, _expected(pools, table, rows, n, q, 128 ** -0.5))
    n.copy_(full)
    lanes = [(torch.cuda.Stream(), ops.kv4_decode_workspace(4, 8, 2, 128, "cuda"), torch.empty_like(q)) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, w, o in lanes:
            with torch.cuda.stream(stream):
                ops.kv4_decode(q, *pools, table, rows, n, workspace=w, out=o)
    torch.cuda.synchronize()
    assert torch.equal(lanes[0][2], lanes[1][2])
    _near(lanes[0][2], _expected(pools, table, rows, n, q, 128 ** -0.5))


@pytest.mark.parametrize("dim", DIMS)
def test_numbers_far_from_one(dim):
    """Queries, keys and values of sizes from 2^-60 to 2^60, one step a thousand times another's."""
    from astrai_b200 import ops

    for qs, ks, vs in ((2.0 ** 40, 2.0 ** -42, 2.0 ** 60), (2.0 ** -60, 2.0 ** 57, 2.0 ** -60), (1e-20, 1e-20, 1e-3), (3.0, 3.0, 2.0 ** 100)):
        pools, table, rows, n, q, _ = _case([70, 40], 4, 2, dim, seed=7)
        q = (q.float() * qs).bfloat16()
        k, v = _rows(110, 2, dim, seed=8).float() * ks, _rows(110, 2, dim, seed=9).float() * vs
        v[::3] *= 1e-3
        used = torch.cat([table[int(r), :m] for r, m in zip(rows, n.tolist())])
        ops.kv4_append_(k.bfloat16(), v.bfloat16(), *pools, used)
        _near(ops.kv4_decode(q, *pools, table, rows, n), _expected(pools, table, rows, n, q, dim ** -0.5))


def test_bad_metadata_is_left_out():
    from astrai_b200 import ops

    pools, table, rows, n, q, new = _case([40, 50, 33, 64], 4, 2, 128, seed=11)
    table[rows[0].long(), 3], table[rows[0].long(), 39] = -1, 2 ** 31 - 1  # slots outside the pool, the last one's among them
    rows[1], n[2], n[3] = 77, 10 ** 12, -4  # a row outside the table; lengths beyond the row and below 0
    out = ops.kv4_decode(q, *pools, table, rows, n, *new)
    n = n.clamp(min=0)
    table[rows[2].long()] = torch.where(table[rows[2].long()] == -5, -1, table[rows[2].long()])
    _near(out, _expected(pools, table, rows, n, q, 128 ** -0.5))
    assert not out[1].any() and not out[3].any()


def test_a_poisoned_key_spoils_its_own_request_only():
    from astrai_b200 import ops

    pools, table, rows, n, q, _ = _case([40, 50], 4, 2, 64, seed=12)
    bad = _rows(1, 2, 64, seed=13)
    bad[0, 1, 5] = math.nan
    ops.kv4_append_(bad, _rows(1, 2, 64, seed=14), *pools, table[rows[0].long(), 7:8])
    out = ops.kv4_decode(q, *pools, table, rows, n)
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all() and torch.isfinite(out[1]).all()
    value = _rows(1, 2, 64, seed=15)
    value[0, 0, 40] = math.inf
    ops.kv4_append_(_rows(1, 2, 64, seed=16), value, *pools, table[rows[1].long(), 2:3])
    out = ops.kv4_decode(q, *pools, table, rows, n)
    assert torch.isnan(out[1, :2, 32:]).all() and torch.isfinite(out[1, :2, :32]).all() and torch.isfinite(out[1, 2:]).all()


def test_decode_is_deterministic_replays_and_runs_on_other_streams():
    from astrai_b200 import ops

    lens = [300, 1, 77, 0, 512]
    pools, table, rows, n, q, new = _case(lens, 8, 2, 128, seed=17)
    work = ops.kv4_decode_workspace(5, 8, 2, 128, "cuda")
    first = ops.kv4_decode(q, *pools, table, rows, n, *new, max_len=512, workspace=work)
    assert torch.equal(first, ops.kv4_decode(q, *pools, table, rows, n, *new, max_len=512, workspace=work))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.kv4_decode(q, *pools, table, rows, n, max_len=512, workspace=ops.kv4_decode_workspace(5, 8, 2, 128, "cuda"))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    graphs = []
    for _ in range(2):  # two graphs with a workspace each
        w, out, g = ops.kv4_decode_workspace(5, 8, 2, 128, "cuda"), torch.empty_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.kv4_decode(q, *pools, table, rows, n, *new, max_len=512, workspace=w, out=out)
        graphs.append((g, out, w))
    q2 = torch.randn_like(q)
    q.copy_(q2)
    n.add_(torch.tensor([-100, 0, -1, 0, -7], device="cuda"))
    graphs[0][0].replay()
    graphs[1][0].replay()
    want = _expected(pools, table, rows, n, q, 128 ** -0.5)
    for _, out, _ in graphs:
        _near(out, want)


def test_slots_beyond_two_gigabytes():
    """A pool whose codes pass 2^31 bytes: the rows at its end."""
    from astrai_b200 import ops

    slots, heads, dim = 2 ** 21 + 64, 8, 256  # 2.1 G bytes of codes
    pools = _pools(slots, heads, dim)
    at = torch.arange(slots - 40, slots, device="cuda")
    k, v = _rows(40, heads, dim, seed=18), _rows(40, heads, dim, seed=19)
    ops.kv4_append_(k, v, *pools, at)
    table = at.int().view(1, 40)
    n, rows = torch.tensor([40], device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    q = _rows(1, heads, dim, seed=20)
    _near(ops.kv4_decode(q, *pools, table, rows, n), _expected(pools, table, rows, n, q, dim ** -0.5))
    gk, _ = ops.kv4_gather(*pools, at)
    assert (gk.float() - k.float()).abs().max() < 1.0
    paged = [t.view(1, slots, heads, -1) for t in pools]
    ops.copy_pages_(paged, [slots // 16 - 1], [3], 16)
    assert torch.equal(pools[0][48:64], pools[0][slots - 16:])


def test_decode_refusals():
    from astrai_b200 import ops

    pools, table, rows, n, q, new = _case([20, 9], 4, 2, 64, seed=21)
    ok = dict(q=q, k_codes=pools[0], k_meta=pools[1], v_codes=pools[2], v_meta=pools[3], req_to_token=table, req_pool_indices=rows, seq_lens=n)
    wrong = [dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.repeat(1, 5, 1)), dict(seq_lens=n.int()), dict(seq_lens=n[:1]),
             dict(req_pool_indices=rows.long()), dict(req_to_token=table.long()), dict(req_to_token=table.t()), dict(k_codes=pools[0][:, :1]),
             dict(k_meta=pools[1].float()), dict(v_codes=pools[2].cpu()), dict(k_new=new[0]), dict(k_new=new[0].float(), v_new=new[1]),
             dict(k_new=new[0][:1], v_new=new[1][:1]), dict(out=q.float()), dict(out=q[:1]),
             dict(workspace=ops.kv4_decode_workspace(1, 4, 2, 64, "cuda")), dict(workspace=ops.kv4_decode_workspace(2, 4, 2, 64, "cuda", parts=1)), dict(workspace=ops.kv4_decode_workspace(2, 4, 2, 128, "cuda")),
             dict(req_to_token=table[:0]), dict(out=torch.empty(q.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(q.shape))]
    for bad in wrong:
        with pytest.raises(RuntimeError, match="kv4_decode"):
            ops.kv4_decode(**{**ok, **bad})
    loc = torch.arange(2, device="cuda")
    for args in ((new[0].float(), new[1], *pools, loc), (*new, *pools, loc[:1]), (*new, *pools, loc.float()), (*new, *pools, loc.cpu()),
                 (new[0], new[1][:1], *pools, loc)):
        with pytest.raises(RuntimeError, match="kv4_append_"):
            ops.kv4_append_(*args)
    with pytest.raises(RuntimeError, match="kv4_gather"):
        ops.kv4_gather(*pools, loc[:, None])
    assert ops.kv4_decode(**{**ok, "q": q[:0], "req_pool_indices": rows[:0], "seq_lens": n[:0]}).shape == (0, 4, 64)


# ---------------------------------------------------------------------------------------------------------- page copies
@pytest.mark.parametrize("page,inner,dtype", [(16, (4, 64), torch.uint8), (1, (3,), torch.uint8), (8, (2, 2, 2), torch.bfloat16), (3, (1, 2), torch.float16), (5, (1,), torch.float32)])
def test_copy_pages(page, inner, dtype):
    from astrai_b200 import ops

    g = torch.Generator().manual_seed(page)
    pages, layers = 700, 3
    pools = [torch.randint(0, 100, (layers, pages * page + 2, *inner), generator=g).to(dtype).cuda(),
             torch.randn(layers, pages * page + 2, 1, generator=g).cuda()]
    order = torch.randperm(pages, generator=g).tolist()
    for n in (1, 300):
        want = [p.clone() for p in pools]
        src, dst = [order[0]] + order[:n - 1], order[n:2 * n]
        ops.copy_pages_(pools, src, dst, page)
        at = torch.arange(pages * page + 2)
        for s, d in zip(src, dst):
            at[d * page:(d + 1) * page] = torch.arange(s * page, (s + 1) * page)
        for p, w in zip(pools, want):
            assert torch.equal(p, w[:, at.cuda()])
    before = [p.clone() for p in pools]
    for src, dst in (([0], [pages + 2]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1, 2])):
        with pytest.raises(ValueError, match="copy_pages_"):
            ops.copy_pages_(pools, src, dst, page)
    assert all(torch.equal(p, b) for p, b in zip(pools, before))


# -------------------------------------------------------------------------------------------- the operators as used
def _model(**over):
    from astrai_b200.config import AutoRegressiveLMConfig
    from astrai_b200.models import AutoRegressiveLM

    torch.manual_seed(0)
    cfg = AutoRegressiveLMConfig(**{**dict(vocab_size=512, hidden_size=512, num_hidden_layers=2, rms_norm_eps=1e-6, intermediate_size=512,
                                           tie_word_embeddings=True, max_position_embeddings=512, rope_theta=10000.0,
                                           num_attention_heads=4, num_key_value_heads=2), **over})
    return AutoRegressiveLM(cfg).to("cuda", torch.bfloat16).eval()


class _Tok:
    stop_ids = []

    def decode(self, ids, skip_special_tokens=True):
        return " ".join(map(str, ids))


@pytest.mark.parametrize("fwd,dim", [("prefill", 64), ("prefill", 128), ("prefill", 32), ("decode", 128), ("decode", 256)])
def test_cached_attention_over_a_four_bit_cache(fwd, dim):
    """``ops.attention`` as the models call it, against 64-bit attention on what the cache holds.  Prefill rounds keys and
    values to bf16 (2^-8 of each: 2^-8 sum p |v|, and the logits by 2^-8 sum |q k| - bounded here through their spread) and
    the flash kernel its probabilities (2^-8 sum p |v|)."""
    from astrai_b200 import ops
    from astrai_b200.inference.cache import PagePool, TaskCacheManager
    from astrai_b200.inference.workspace import InferenceWorkspace
    from astrai_b200.ops import kv4

    lens, cached = [70, 33, 129], [0, 16, 100]
    heads, kv_heads = 4, 2
    pool = PagePool(2, kv_heads, dim, 4, 256, "cuda", torch.bfloat16, page_size=16, n_tokens=1024, kv_dtype="int4")
    tc = TaskCacheManager(pool)
    ws = InferenceWorkspace(4, 256, heads, dim, "cuda", torch.bfloat16, n_kv_heads=kv_heads, max_prefill_tokens=512)
    ids = [f"t{i}" for i in range(3)]
    for t, n in zip(ids, lens):
        assert tc.task_alloc(t, [hash((t, j)) % 1000 for j in range(n)])
    st = pool.storage
    everything = torch.arange(1024, device="cuda")
    k_all, v_all = _rows(1024, kv_heads, dim, seed=31), _rows(1024, kv_heads, dim, seed=32)
    ops.kv4_append_(k_all, v_all, st.k_buffer[1], st.k_meta[1], st.v_buffer[1], st.v_meta[1], everything)
    starts = cached if fwd == "prefill" else [n - 1 for n in lens]
    counts = [n - s for n, s in zip(lens, starts)]
    kv = tc.bind(ids, ws, start_positions=starts) if fwd == "prefill" else tc.bind(ids, ws)
    q = _rows(sum(counts), heads, dim, seed=33)
    k, v = _rows(sum(counts), kv_heads, dim, seed=34), _rows(sum(counts), kv_heads, dim, seed=35)
    out = ops.attention(q, k, v, kv, 1, None, True, fwd)
    assert not st.k_buffer[0].any()  # the other layer is left alone
    start = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        slots = kv.req_to_token[int(kv.req_pool_indices[i]), :n].long()
        kd, vd = (kv4.dequantize(b[1][slots], m[1][slots], keys).double() for b, m, keys in
                  ((st.k_buffer, st.k_meta, True), (st.v_buffer, st.v_meta, False)))
        want_k = kv4.dequantize(*kv4.quantize(k[start:start + c].cpu(), True), True).double().cuda()
        assert torch.equal(kd[n - c:], want_k)
        kd, vd = (x.repeat_interleave(2, 1) for x in (kd, vd))
        qd = q[start:start + c].double()
        logit = torch.einsum("shd,lhd->hsl", qd, kd) * dim ** -0.5
        size = torch.einsum("shd,lhd->hsl", qd.abs(), kd.abs()) * dim ** -0.5
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - c, n, device="cuda")[:, None]
        p = torch.softmax(logit.masked_fill(~seen, -math.inf), -1)
        o = torch.einsum("hsl,lhd->shd", p, vd)
        mean_v = torch.einsum("hsl,lhd->shd", p, vd.abs())
        # rounded keys move a logit by at most 2^-8 of `size`; p then changes by twice that, relatively
        moved = torch.einsum("hsl,lhd->shd", p * size * 2.0 ** -8 * 2, vd.abs()) + 2 * 2.0 ** -8 * mean_v * (p * size).sum(-1).t()[..., None]
        tol = 2.0 ** -8 * o.abs() + 3 * 2.0 ** -8 * mean_v + moved
        assert ((out[start:start + c].double() - o).abs() <= tol).all()
        start += c


def test_serving_run_with_graphs_forks_and_chunks():
    """Store, read, prefill, decode and page copies together: greedy answers through captured decode graphs, through eager
    launches and as forks of one prefilled prompt."""
    from astrai_b200.inference import InferenceScheduler
    from astrai_b200.ops import native

    model = _model()
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(5, 500, (n,), generator=g).tolist() for n in (40, 3, 65, 130)]
    kw = dict(max_batch_size=8, max_seq_len=256, kv_dtype="int4")
    eager = InferenceScheduler(model, _Tok(), enable_cuda_graph=False, **kw).run_batch(prompts, max_tokens=12, temperature=0.0)
    sched = InferenceScheduler(model, _Tok(), enable_cuda_graph=True, **kw)
    assert sched.cuda_graph_enabled
    graphed = sched.run_batch(prompts, max_tokens=12, temperature=0.0)
    assert all(len(a) == 12 for a in eager + graphed)
    # padded batch buckets and split counts differ, so sums may round otherwise: the first token is the prefill's, equal
    assert [a[0] for a in eager] == [a[0] for a in graphed]
    forked = sched.run_batch(prompts[:2], max_tokens=12, temperature=0.0, samples_per_prompt=3)
    assert all(len(a) == 12 for a in forked)
    assert native.kernel_status("cuda") == 0


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("gap", [0, 12, 20, 26, 30, 34, 40, 60])
def test_ranges_inside_a_tile_and_a_head(gap, dim):
    """Steps of one group 2^gap below another's, and query numbers 2^gap below the head's largest with keys as far above.

    ``p s`` is rounded to fp16 after scaling by one power of two a tile: 2^-11 of it while it is at least 2^-28 of the tile's
    largest step S, else half of fp16's smallest number over a scale of at least 2^14 / S: 2^-25 2^-14 S = 2^-39 S, times a
    code of at most 15.  The weights are relative to the largest so far, so a key's share of the normalised result is off by
    15 x 2^-39 S at most, n keys' by n times that.  A query number keeps its 8 bits while its lowest one is at least 2^-24
    after scaling by at least 2^13 over the largest number Q, and over 16 at odd positions: down to 2^-26 Q.  Below, it is off
    by 16 x 2^-25 x 2^-13 Q = 2^-34 Q, times a code of at most 15 and the step."""
    from astrai_b200 import ops
    from astrai_b200.ops import kv4

    pools, table, rows, n, q, _ = _case([70, 40, 300], 4, 2, dim, seed=41)
    used = torch.cat([table[int(r), :m] for r, m in zip(rows, n.tolist())])
    scale = dim ** -0.5
    far = torch.ones(dim, device="cuda")
    far[32:64] = 2.0 ** -gap
    k, v = _rows(410, 2, dim, seed=42), _rows(410, 2, dim, seed=43)
    for kk, vv, qq, short in ((k, v * far, q, "value"), (k / far, v, q * far, "query")):
        kk, vv, qq = (x.bfloat16() for x in (kk, vv, qq))
        ops.kv4_append_(kk, vv, *pools, used)
        o, tol = _expected(pools, table, rows, n, qq, scale)
        out = ops.kv4_decode(qq, *pools, table, rows, n)
        for i, length in enumerate(n.tolist()):
            slots = table[int(rows[i]), :length].long()
            if short == "value":
                largest = pools[3][slots][..., 1].double().amax((0, 2)).repeat_interleave(2)  # of a kv head -> [heads]
                tol[i] += length * 15 * 2.0 ** -39 * largest[:, None]
            else:
                steps = (pools[1][slots][..., 1].double().sum(-1) * 32).amax(0).repeat_interleave(2)  # sum over a row's numbers
                off = 15 * 2.0 ** -34 * qq[i].double().abs().amax(-1) * steps * scale
                vd = kv4.dequantize(pools[2][slots], pools[3][slots], False).double().abs().amax(0).repeat_interleave(2, 0)
                tol[i] += 2 * (off.exp() - 1).clamp(max=1)[:, None] * vd  # p changes by a factor of at most exp(off), its sum too
        _near(out, (o, tol))
