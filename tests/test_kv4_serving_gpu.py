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


# --------------------------------------------------------------------------------------------- what serving runs
def _scheduler(model, **kw):
    from astrai_b200.inference import InferenceScheduler
    from test_kv4_gpu import _Tok

    return InferenceScheduler(model, _Tok(), **{"max_batch_size": 8, "max_seq_len": 256, "kv_dtype": "int4", **kw})


def _record_logits(sched, monkeypatch):
    """Every row of logits that is sampled from, ``(task id, position in the answer, logits)`` in order."""
    seen, plain = [], sched._executor._sample

    def sample(logits, tasks, *args, **kw):
        seen.extend((t.task_id, len(t.output_ids), row.float().clone()) for t, row in zip(tasks, logits))
        return plain(logits, tasks, *args, **kw)

    monkeypatch.setattr(sched._executor, "_sample", sample)
    return seen


PROMPTS = [[(7 * i + 3 * j * j) % 490 + 5 for j in range(n)] for i, n in enumerate((40, 3, 65, 130, 16))]


@pytest.mark.parametrize("paged", [True, False])
def test_a_replayed_step_with_padded_rows_computes_what_the_cache_holds(paged, monkeypatch):
    """A decode step of 5 requests in a graph of 8 rows: its logits are those of the same launches made one by one, and the
    attention of every layer is the 64-bit one over the rows that the cache holds."""
    from astrai_b200.ops import kv4
    from test_kv4_gpu import _expected as expected, _model, _near

    sched = _scheduler(_model(), paged=paged, page_size=16 if paged else 1)
    ex, tc = sched._executor, sched._task_cache
    assert sched.cuda_graph_enabled and ex._bucket(5) == 8
    from astrai_b200.inference.task import Task

    tasks = [Task(f"t{i}", list(p), 9, 0.0, 1.0, 50, 0.0, 64) for i, p in enumerate(PROMPTS)]
    for t in tasks:
        t.input_tokens = len(t.prompt_ids)
        assert tc.task_alloc(t.task_id, t.prompt_ids)
    done, tokens = ex.execute_prefill(tasks)
    assert done == tasks
    for t, token in zip(tasks, tokens):
        t.output_ids.append(token)
        t.mark_prefill_done()
    calls, plain = [], kv4.kv4_decode

    def recorded(q, *args, **kw):
        out = plain(q, *args, **kw)
        calls.append((q.clone(), args, out.clone(), kw["max_len"]))
        return out

    for step in range(3):
        for t in tasks:
            assert tc.task_extend(t.task_id, t.next_pos)
        got = []
        with monkeypatch.context() as patch:
            patch.setattr(ex, "_sample", lambda logits, *a, **kw: got.append(logits.clone()) or logits.argmax(-1).tolist())
            tokens = ex.execute_decode(tasks)  # the graph
        ws = ex.workspace
        with monkeypatch.context() as patch, torch.inference_mode():
            patch.setattr(kv4, "kv4_decode", recorded)
            kv = ex._padded(tc.bind([t.task_id for t in tasks], ws), 5, 8)  # the same step once more, launch by launch
            ex._zero_padding(5, 8)
            out = ex.model(input_ids=ws.input_ids[:8], kv_cache=kv, position_ids=ws.position_ids[:8], fwd="decode")["logits"]
        assert torch.equal(got[0], out[:5])
        lens = torch.tensor([len(p) + 1 + step for p in PROMPTS] + [0] * 3)
        assert len(calls) == 2 * (step + 1)
        for q, (*pools, table, rows, n), o, max_len in calls[-2:]:
            assert torch.equal(n.cpu(), lens) and max_len == 256
            _near(o, expected(pools, table, rows, n, q, q.shape[-1] ** -0.5))
        ex._decode_cache = None  # the bind in between was not the executor's
        for t, token in zip(tasks, tokens):
            t.output_ids.append(token)
            t.advance_kv()


@pytest.mark.parametrize("kv_dtype", ["int4", "auto"])
@pytest.mark.parametrize("paged", [True, False])
def test_a_fork_holds_its_leaders_rows_in_every_layer(paged, kv_dtype):
    from test_kv4_gpu import _model

    sched = _scheduler(_model(), paged=paged, page_size=16 if paged else 1, kv_dtype=kv_dtype, enable_cuda_graph=False)
    tc, table, pools = sched._task_cache, sched.cache.req_pool.req_to_token, sched.cache.storage.pools()
    assert tc.task_alloc("a", list(range(100)))
    for t in pools:
        t.copy_(torch.randint(1, 100, t.shape, device="cuda"))
    before = [t.clone() for t in pools]
    for name, length in (("b", 100), ("c", 37), ("d", 32), ("e", 1)):
        assert tc.task_fork("a", name, length)
        a, f = (table[tc.state(n).req_idx, :length].long() for n in ("a", name))
        assert (a.device.type, a.numel()) == ("cuda", length)
        for t, old in zip(pools, before):
            assert torch.equal(t[:, f], old[:, a]) and torch.equal(t[:, a], old[:, a])
        shared = length // 16 * 16 if paged else 0
        assert torch.equal(a[:shared], f[:shared]) and not set(a[shared:].tolist()) & set(f[shared:].tolist())


def _close(a, b, what):
    """Logits of the same numbers through launches of other shapes.  Both runs round to bf16 (2^-9 of a number, either way)
    after some 10 operations in each of 2 layers and may round each the other way: 20 x 2^-8 of the logits' size if every
    rounding adds up; the prompt's last position sees bf16 rows in one and the codes' own numbers in the other: 2^-8 more in
    keys and values of each layer.  That is 0.1; a wrong row, page or length gives logits of another token, 1.4."""
    off = ((a - b).norm() / b.norm()).item()
    assert off < 0.1, f"{what}: {off:.3f}"


def test_forks_answer_from_their_leaders_prompt(monkeypatch):
    from test_kv4_gpu import _model

    sched = _scheduler(_model(), max_batch_size=16)
    names = {}
    plain = sched._task_cache.task_fork
    monkeypatch.setattr(sched._task_cache, "task_fork", lambda a, b, n=None: names.update({b: a}) or plain(a, b, n))
    seen = _record_logits(sched, monkeypatch)
    answers = sched.run_batch(PROMPTS, max_tokens=6, temperature=0.0, samples_per_prompt=3)
    assert len(answers) == 15 and all(len(a) == 6 for a in answers) and len(names) == 10
    first = {task: row for task, n, row in seen if n == 0}
    for fork, leader in names.items():
        _close(first[fork], first[leader], f"{fork} of {leader}")
    leaders = list(dict.fromkeys(names.values()))
    for i, a in enumerate(leaders):  # the bound tells prompts apart
        for b in leaders[:i]:
            assert ((first[a] - first[b]).norm() / first[b].norm()).item() > 0.3


@pytest.mark.parametrize("kv_dtype", ["int4", "auto"])
def test_chunks_answer_as_the_whole_prompt_does(kv_dtype, monkeypatch):
    from test_kv4_gpu import _model

    model, rows = _model(), []
    for kw in ({}, {"chunked_prefill": True, "max_prefill_tokens": 24}):
        sched = _scheduler(model, kv_dtype=kv_dtype, **kw)
        seen = _record_logits(sched, monkeypatch)
        for p in PROMPTS:  # one after the other: a request's logits come in order
            assert len(sched.run_batch([p], max_tokens=1, temperature=0.0)[0]) == 1
        assert len(seen) == len(PROMPTS)
        rows.append([row for _, _, row in seen])
    for p, whole, cut in zip(PROMPTS, *rows):
        _close(cut, whole, f"prompt of {len(p)}")


@pytest.mark.parametrize("counts", [[5, 3], [1, 1]])
def test_no_derivative_is_dropped_on_the_way_through_a_four_bit_cache(counts):
    import torch.autograd.forward_ad as fwAD

    from astrai_b200 import ops

    heads, kv_heads, dim, lens = 4, 2, 64, [70, 40]
    pool, tc, ws = _cached(lens, heads, kv_heads, dim)
    kv = tc.bind(["t0", "t1"], ws, start_positions=[n - c for n, c in zip(lens, counts)])
    q, k, v = (_rows(sum(counts), h, dim, seed=50 + h) for h in (heads, kv_heads, kv_heads))
    plain = ops.attention(q, k, v, kv, 0, None, True, "prefill")
    qg = q.clone().requires_grad_()
    out = ops.attention(qg, k, v, kv, 0, None, True, "prefill")
    o, tol = _expected(pool, kv, q, counts, lens, 1, dim ** -0.5)
    for got in (plain, out.detach()):
        assert ((got[counts[0]:].double() - o).abs() <= tol).all()
    out.float().sum().backward()
    assert torch.isfinite(qg.grad).all() and qg.grad.abs().max() > 0
    with fwAD.dual_level():
        try:
            out = ops.attention(fwAD.make_dual(q, torch.randn_like(q)), k, v, kv, 0, None, True, "prefill")
        except (NotImplementedError, RuntimeError):
            return
        assert fwAD.unpack_dual(out).tangent is not None
