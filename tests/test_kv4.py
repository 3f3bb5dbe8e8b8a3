"""The 4-bit KV cache on the CPU: format, rows in and out, decode attention, page copies, serving over it, forks."""

import math

import pytest
import torch

from helpers import tiny_config

DIMS = (32, 64, 128, 256)


def _pools(slots, heads, dim, layers=None, device="cpu"):
    lead = (slots, heads) if layers is None else (layers, slots, heads)
    return [t for _ in "kv" for t in (torch.zeros(*lead, dim // 2, dtype=torch.uint8, device=device),
                                      torch.zeros(*lead, dim // 32, 2, dtype=torch.bfloat16, device=device))]


class _Tok:
    stop_ids = []

    def decode(self, ids, skip_special_tokens=True):
        return " ".join(map(str, ids))


@pytest.fixture(scope="module")
def model():
    from astrai_b200.models import AutoRegressiveLM

    torch.manual_seed(0)  # heads of 32: the narrowest that a 4-bit cache holds
    return AutoRegressiveLM(tiny_config(hidden_size=64, intermediate_size=96, num_attention_heads=2, num_key_value_heads=1)).eval()


def _scheduler(model, **kw):
    from astrai_b200.inference import InferenceScheduler

    return InferenceScheduler(model, _Tok(), **{"max_batch_size": 8, "max_seq_len": 48, "page_size": 4, "kv_dtype": "int4", **kw})


# ------------------------------------------------------------------------------------------------------------- format
@pytest.mark.parametrize("keys", [True, False])
@pytest.mark.parametrize("dim", DIMS)
def test_packing_is_a_permutation(dim, keys):
    from astrai_b200.ops import kv4

    codes = torch.randint(0, 16, (3, 2, dim), dtype=torch.uint8)
    data = kv4.pack(codes, keys)
    assert data.shape == (3, 2, dim // 2) and torch.equal(kv4.unpack(data, keys), codes)
    # one number at a time: each has a half byte of its own
    eye = kv4.unpack(kv4.pack(torch.eye(dim, dtype=torch.uint8), keys), keys)
    assert torch.equal(eye, torch.eye(dim, dtype=torch.uint8))


@pytest.mark.parametrize("offset,width", [(0.0, 1.0), (3.0, 0.01), (-1e4, 1e-2), (1e-30, 1e-30), (0.0, 1e30)])
def test_a_number_is_off_by_half_a_step_and_the_middle_s_rounding(offset, width):
    from astrai_b200.ops import kv4

    torch.manual_seed(1)
    x = (torch.randn(40, 3, 128) * width + offset).bfloat16()
    codes, meta = kv4.quantize(x, True)
    m, s = meta[..., 0].double(), meta[..., 1].double()
    off = (kv4.dequantize(codes, meta, True).double() - x.double()).abs().unflatten(-1, (-1, 32)).amax(-1)
    # half a step; the middle's rounding (2^-8 of it), which can also push an end of the group over the last code; the
    # step's rounding (2^-8 of it) over 8 codes; the fp32 sum of the read-back
    bound = s / 2 + 2 ** -8 * m.abs() + 8 * 2 ** -8 * s + 2 ** -22 * (m.abs() + 8 * s)
    assert (off <= bound).all()


def test_special_groups():
    from astrai_b200.ops import kv4

    x = torch.zeros(7, 1, 32, dtype=torch.bfloat16)
    x[0] = 1.2345
    x[1, 0, 3] = math.inf
    x[2, 0, 0] = math.nan
    x[3, 0, :2] = torch.tensor([2.0 ** 119, -2.0 ** 119])  # spreads over 2^120
    x[4, 0, 1] = 2.0 ** -126                               # a step below 2^-120
    x[5] = torch.tensor([1.0, -1.0] * 16)
    back = kv4.dequantize(*kv4.quantize(x, True), True)
    assert torch.equal(back[0], x[0].float()) and (back[4] == 0).all()
    assert all(torch.isnan(back[i]).all() for i in (1, 2, 3))
    assert torch.isfinite(back[5]).all() and (back[5] - x[5].float()).abs().max() <= 1 / 15 + 8 * 2 ** -8 * 2 / 15 + 2 ** -8


# ------------------------------------------------------------------------------------------------------ rows in and out
@pytest.mark.parametrize("loc_dtype", [torch.int32, torch.int64])
def test_rows_go_where_they_belong(loc_dtype):
    from astrai_b200 import ops
    from astrai_b200.ops import kv4

    torch.manual_seed(2)
    pools = _pools(10, 2, 64)
    k, v = torch.randn(5, 2, 64).bfloat16(), torch.randn(5, 2, 64).bfloat16()
    loc = torch.tensor([7, -1, 0, 10, 3], dtype=loc_dtype)  # two slots outside the pool: skipped, read as zeros
    ops.kv4_append_(k, v, *pools, loc)
    assert not pools[0][[1, 2, 4, 5, 6, 8, 9]].any() and not pools[3][[1, 2, 4, 5, 6, 8, 9]].any()
    gk, gv = ops.kv4_gather(*pools, loc)
    for got, x, keys in ((gk, k, True), (gv, v, False)):
        want = kv4.dequantize(*kv4.quantize(x, keys), keys).bfloat16()
        want[[1, 3]] = 0
        assert got.dtype == torch.bfloat16 and torch.equal(got, want)
    ops.kv4_append_(k[:0], v[:0], *pools, loc[:0])
    assert ops.kv4_gather(*pools, loc[:0])[0].shape == (0, 2, 64)


def _softmax_attention(q, k, v, scale):
    """q [Hq, D], k / v [L, Hkv, D] in 64 bits."""
    group = q.shape[0] // k.shape[1]
    out = []
    for h in range(q.shape[0]):
        p = torch.softmax(k[:, h // group].double() @ q[h].double() * scale, 0)
        out.append(p @ v[:, h // group].double())
    return torch.stack(out)


@pytest.mark.parametrize("store", [False, True])
def test_decode_attention_statement(store):
    from astrai_b200 import ops
    from astrai_b200.ops import kv4

    torch.manual_seed(3)
    pools = _pools(64, 2, 32)
    ops.kv4_append_(torch.randn(64, 2, 32).bfloat16(), torch.randn(64, 2, 32).bfloat16(), *pools, torch.arange(64))
    table = torch.randperm(60).int().view(5, 12)
    table[2, 1], table[2, 4] = -1, 64  # left out
    lens = torch.tensor([12, 0, 7, 1, 99])  # the last one is cut to the row
    rows = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32)
    q = torch.randn(5, 6, 32)
    new = (torch.randn(5, 2, 32).bfloat16(), torch.randn(5, 2, 32).bfloat16()) if store else (None, None)
    out = ops.kv4_decode(q, *pools, table, rows, lens, *new)
    for i, n in enumerate([12, 0, 7, 1, 12]):
        if n == 0:
            assert not out[i].any()
            continue
        slots = table[i, :n].long()
        slots = slots[(slots >= 0) & (slots < 64)]
        k, v = kv4.dequantize(pools[0][slots], pools[1][slots], True), kv4.dequantize(pools[2][slots], pools[3][slots], False)
        if store:
            assert torch.equal(k[-1], kv4.dequantize(*kv4.quantize(new[0][i], True), True))
        assert torch.allclose(out[i].double(), _softmax_attention(q[i], k, v, 32 ** -0.5), atol=1e-5)
    with pytest.raises(ValueError, match="together"):
        ops.kv4_decode(q, *pools, table, rows, lens, k_new=q[:, :2])
    with pytest.raises(ValueError, match="heads"):
        ops.kv4_decode(q[:, :5], *pools, table, rows, lens)


# ---------------------------------------------------------------------------------------------------------- page copies
def test_copy_pages():
    from astrai_b200 import ops

    pools = [torch.randint(0, 255, (2, 23, 3), dtype=torch.uint8), torch.randn(2, 23, 2, 2)]
    before = [p.clone() for p in pools]
    ops.copy_pages_(pools, [0, 0, 3], [2, 1, 4], 4)  # a source may serve twice; three slots behind the last page stay
    for p, b in zip(pools, before):
        assert torch.equal(p, torch.cat([b[:, :4], b[:, :4], b[:, :4], b[:, 12:16], b[:, 12:16], b[:, 20:]], dim=1))
    ops.copy_pages_(pools, [], [], 4)


@pytest.mark.parametrize("src,dst,page,match", [
    ([0], [4], 4, "outside"), ([-1], [0], 4, "outside"), ([0, 1], [2, 2], 4, "twice"), ([0, 1], [1, 2], 4, "read and written"),
    ([0], [0], 4, "read and written"), ([0], [1, 2], 4, "as many"), ([0], [1], 0, "page_size"),
])
def test_copy_pages_refusals(src, dst, page, match):
    from astrai_b200 import ops

    pool = torch.arange(32.0).view(2, 16)
    before = pool.clone()
    with pytest.raises(ValueError, match=match):
        ops.copy_pages_([pool], src, dst, page)
    with pytest.raises(ValueError, match="pools"):
        ops.copy_pages_([], [0], [1], 4)
    with pytest.raises(RuntimeError, match="as many"):
        ops.copy_pages_([pool, pool[:, :8].contiguous()], [0], [1], 4)
    assert torch.equal(pool, before)


# ------------------------------------------------------------------------------------------------------------- serving
def test_pool_refusals():
    from astrai_b200.inference.cache import PagePool

    with pytest.raises(ValueError, match="kv_dtype"):
        PagePool(1, 1, 64, 2, 16, "cpu", torch.float32, kv_dtype="int3")
    with pytest.raises(ValueError, match="head_dim"):
        PagePool(1, 1, 96, 2, 16, "cpu", torch.float32, kv_dtype="int4")
    with pytest.raises(ValueError, match="bf16"):
        PagePool(1, 1, 64, 2, 16, "cuda", torch.float16, kv_dtype="int4")
    pool = PagePool(3, 2, 64, 2, 16, "cpu", torch.float32, page_size=4, n_tokens=32, kv_dtype="int4")
    bits = sum(t.numel() * t.element_size() for t in pool.storage.pools()) * 8
    assert bits == 5 * 2 * 3 * 32 * 2 * 64  # five bits a number


def test_greedy_answers_do_not_depend_on_chunks_mates_or_layout(model):
    prompts = [list(range(5, 25)), list(range(9, 12)), [7], list(range(100, 131))]
    want = [_scheduler(model).run_batch([p], max_tokens=9, temperature=0.0)[0] for p in prompts]
    assert all(len(w) == 9 for w in want)
    for kw in ({}, {"chunked_prefill": True, "max_prefill_tokens": 5}, {"page_size": 1, "paged": False}, {"page_size": 16}):
        assert _scheduler(model, **kw).run_batch(prompts, max_tokens=9, temperature=0.0) == want, kw


def test_four_bits_stay_near_full_precision(model):
    """One forward over a cached prompt: the logits' change is the size that the rows' change explains (the cache's rows are
    off by about a tenth of their spread), not a different function."""
    from astrai_b200.inference.cache import PagePool, TaskCacheManager
    from astrai_b200.inference.workspace import InferenceWorkspace

    cfg, prompt, logits = model.config, list(range(30, 50)), {}
    for kind in ("auto", "int4"):
        pool = PagePool.for_model(cfg, 2, 48, "cpu", torch.float32, page_size=4, kv_dtype=kind)
        tc, ws = TaskCacheManager(pool), InferenceWorkspace(2, 48, cfg.num_attention_heads, 32, "cpu", torch.float32)
        assert tc.task_alloc("a", prompt)
        with torch.inference_mode():
            out = model(torch.tensor(prompt), position_ids=torch.arange(20), kv_cache=tc.bind(["a"], ws, start_pos=0), fwd="prefill")
        logits[kind] = out["logits"]
    cos = torch.nn.functional.cosine_similarity(logits["auto"], logits["int4"], dim=-1)
    assert cos.min() > 0.98 and not torch.equal(logits["auto"], logits["int4"])


# --------------------------------------------------------------------------------------------------------------- forks
@pytest.mark.parametrize("kv_dtype", ["auto", "int4"])
@pytest.mark.parametrize("length", [0, 3, 4, 8, 10, 11])
def test_a_fork_goes_its_own_way(length, kv_dtype):
    from astrai_b200.inference.cache import PagePool, TaskCacheManager

    pool = PagePool(2, 1, 32, 4, 32, "cpu", torch.float32, page_size=4, n_tokens=64, kv_dtype=kv_dtype)
    tc = TaskCacheManager(pool)
    free = pool.allocator.available()
    assert tc.task_alloc("a", list(range(11)))
    gen = torch.Generator().manual_seed(length)
    for t in pool.storage.pools():
        t.copy_(torch.randint(0, 100, t.shape, generator=gen))
    assert tc.task_fork("a", "b", length)
    a, b = tc.state("a"), tc.state("b")
    assert b.length == b.cached == length and b.pages[:length // 4] == a.pages[:length // 4]
    assert set(b.pages[length // 4:]).isdisjoint(a.pages)
    table = pool.req_pool.req_to_token
    for t in pool.storage.pools():
        assert torch.equal(t[:, table[a.req_idx, :length].long()], t[:, table[b.req_idx, :length].long()])
    for pos in range(length, 14):  # the fork fills positions of its own; nothing of the first task's changes
        assert tc.task_extend("b", pos)
    mine = table[b.req_idx, length:14].long()
    assert not set(mine.tolist()) & set(table[a.req_idx, :11].tolist())
    tc.task_free("a")
    for t in pool.storage.pools():
        assert t[:, table[b.req_idx, :length].long()].shape[1] == length
    tc.task_free("b")
    assert pool.allocator.available() == free


def test_fork_refusals_and_no_room():
    from astrai_b200.inference.cache import PagePool, TaskCacheManager

    pool = PagePool(1, 1, 32, 3, 16, "cpu", torch.float32, page_size=4, n_tokens=12, kv_dtype="int4")
    tc = TaskCacheManager(pool)
    assert tc.task_alloc("a", list(range(10)))
    with pytest.raises(KeyError):
        tc.task_fork("x", "b")
    with pytest.raises(ValueError, match="exists"):
        tc.task_fork("a", "a")
    for bad in (-1, 11):
        with pytest.raises(ValueError, match="length"):
            tc.task_fork("a", "b", bad)
    assert not tc.task_fork("a", "b")  # no page left for the part of a page
    assert tc.state("b") is None and tc.task_fork("a", "b", 8) and tc.task_fork("a", "c", 4)
    assert not tc.task_fork("a", "d", 4)  # no row left
    for t in "abc":
        tc.task_free(t)
    assert pool.allocator.available() == 3 and len(pool.req_pool.free_slots) == 3


def test_contiguous_rows_fork_by_copy():
    from astrai_b200.inference.cache import PagePool, TaskCacheManager

    pool = PagePool(2, 1, 32, 2, 16, "cpu", torch.float32)
    tc = TaskCacheManager(pool)
    tc.task_alloc("a", [1, 2, 3])
    pool.storage.k_buffer.normal_()
    assert tc.task_fork("a", "b", 2)
    table = pool.req_pool.req_to_token.long()
    assert torch.equal(pool.storage.k_buffer[:, table[tc.state("a").req_idx, :2]], pool.storage.k_buffer[:, table[tc.state("b").req_idx, :2]])


@pytest.mark.parametrize("kw", [{}, {"chunked_prefill": True, "max_prefill_tokens": 6}, {"page_size": 1, "paged": False}, {"kv_dtype": "auto"}])
def test_several_answers_of_a_prompt_share_its_prefill(model, kw):
    prompts = [list(range(40, 53)), [5], list(range(60, 68))]
    sched = _scheduler(model, max_batch_size=9, **kw)
    free = len(sched.cache.req_pool.free_slots)
    single = [sched.run_batch([p], max_tokens=6, temperature=0.0)[0] for p in prompts]
    got = sched.run_batch(prompts, max_tokens=6, temperature=0.0, samples_per_prompt=3)
    assert got == [s for s in single for _ in range(3)]
    assert len(sched.cache.req_pool.free_slots) == free
    toks, logps = sched.run_batch([prompts[0]], max_tokens=4, return_logprobs=True, samples_per_prompt=2)[1]
    assert len(toks) == len(logps) == 4
    # no room for every answer: the ones that do not fit are empty, the others complete
    got = sched.run_batch([prompts[0]], max_tokens=3, temperature=0.0, samples_per_prompt=12)
    assert [len(g) for g in got] == [3] * 9 + [0] * 3
    with pytest.raises(ValueError, match="samples_per_prompt"):
        sched.run_batch(prompts, samples_per_prompt=0)


def test_forks_behind_a_large_decode_batch_are_not_lost(model):
    sched = _scheduler(model, max_batch_size=8, prefill_defer_min_batch=2, prefill_defer_steps=3)
    got = sched.run_batch([[5, 6, 7], [8, 9], [11]], max_tokens=6, temperature=0.0, samples_per_prompt=2)
    assert [len(g) for g in got] == [6] * 6 and got[0] == got[1] and got[2] == got[3]


def test_rollouts_can_share_prompts(model):
    from astrai_b200.trainer.rollout import RolloutGenerator

    class Tok(_Tok):
        def apply_chat_template(self, conv, tokenize=True, add_generation_prompt=True):
            ids = [len(m["content"]) + 3 for m in conv] + [4, 5, 6]
            return ids if tokenize else str(ids)

    batch = {"instruction": ["ab", "abcd"]}
    outs = []
    for share in (False, True):
        gen = RolloutGenerator(_scheduler(model), Tok(), max_tokens=5, group_size=3, temperature=0.0, share_prompts=share)
        outs.append(gen.generate(batch))
    assert torch.equal(outs[0].responses, outs[1].responses) and torch.equal(outs[0].response_mask, outs[1].response_mask)


def test_online_training_shares_prompts(tmp_path):
    """The option reaches the scheduler: each prompt of a batch is asked for once, with a group of answers."""
    from astrai_b200.config import TrainConfig
    from astrai_b200.inference.scheduler import InferenceScheduler
    from astrai_b200.trainer import Trainer
    from helpers import build_tokenizer_dir
    from test_online_training import Instructions, LongerIsBetter, _adamw, _model, collate

    asked, plain = [], InferenceScheduler.run_batch

    def run_batch(self, prompts, **kw):
        asked.append((len(prompts), kw.get("samples_per_prompt", 1)))
        return plain(self, prompts, **kw)

    cfg = dict(strategy="online_grpo", model_fn=_model, dataset=Instructions(), optimizer_fn=_adamw, n_epoch=1, batch_per_device=2,
               grad_accum_steps=1, ckpt_interval=100, random_seed=42, device_type="cpu", backend="gloo", nprocs=1, parallel_mode="none",
               strategy_kwargs={"clip_eps": 0.2, "kl_coef": 0.01, "group_size": 3}, rollout_interval=1, rollout_max_tokens=4,
               reward_model_fn=LongerIsBetter, collate_fn=collate, metrics=["loss"])
    params = build_tokenizer_dir(str(tmp_path / "params"))
    InferenceScheduler.run_batch = run_batch
    try:
        Trainer(TrainConfig(**cfg, ckpt_dir=str(tmp_path / "ck"), rollout_share_prompts=True)).train(param_path=params)
    finally:
        InferenceScheduler.run_batch = plain
    assert asked and all(a == (2, 3) for a in asked)


def test_back_ends_and_caches_that_do_not_fit_are_refused(model):
    from astrai_b200.inference.cache import PagePool
    from astrai_b200.ops import AttentionBackend, attn_backend

    class Own(AttentionBackend):
        def fwd_prefill(self, q, k, v, kv_cache, layer_id, attn_mask=None, is_causal=False):
            from astrai_b200.ops.paged_attention import cached_attention

            with attn_backend("torch_native"):
                return cached_attention(q, k, v, kv_cache, layer_id, attn_mask, is_causal, "prefill")

        fwd_decode = fwd_prefill

    class Reads(Own):
        reads_four_bit = True

    prompt = [list(range(5, 14))]
    want = _scheduler(model).run_batch(prompt, max_tokens=4, temperature=0.0)
    with attn_backend(Own()):
        with pytest.raises(ValueError, match="Own does not read a 4-bit"):
            _scheduler(model).run_batch(prompt, max_tokens=4, temperature=0.0)
        assert _scheduler(model, kv_dtype="auto").run_batch(prompt, max_tokens=4, temperature=0.0)[0]
    with attn_backend(Reads()):
        assert _scheduler(model).run_batch(prompt, max_tokens=4, temperature=0.0) == want
    pool = PagePool.for_model(model.config, 8, 48, "cpu", torch.float32, page_size=4)
    with pytest.raises(ValueError, match="'int4' was asked for"):
        _scheduler(model, cache=pool)
    four = PagePool.for_model(model.config, 8, 48, "cpu", torch.float32, page_size=4, kv_dtype="int4")
    for kw in ({"kv_dtype": "auto"}, {}):  # the cache that was given decides
        assert _scheduler(model, cache=four, **kw).run_batch(prompt, max_tokens=4, temperature=0.0) == want


def test_commands_hand_the_options_on(tmp_path, monkeypatch):
    from click.testing import CliRunner

    from astrai_b200.cli import serve
    from astrai_b200.cli.benchmark import benchmark as bench

    got = {}
    monkeypatch.setattr("astrai_b200.inference.network.app.run_server", lambda **kw: got.update(kw))
    monkeypatch.setattr("astrai_b200.inference.run_server", lambda **kw: got.update(kw), raising=False)
    res = CliRunner().invoke(serve.serve_command, ["--param_path", str(tmp_path), "--kv_dtype", "int4", "--device", "cpu"])
    assert res.exit_code == 0, res.output
    assert got["kv_dtype"] == "int4"
    assert CliRunner().invoke(serve.serve_command, ["--param_path", str(tmp_path), "--kv_dtype", "int3"]).exit_code == 2
    assert all(any(p.name == "kv_dtype" for p in bench.commands[c].params) for c in ("prefill", "decode", "serve"))


def test_histories_are_read_back_in_pieces_of_a_bounded_number_of_keys():
    from astrai_b200.ops.paged_attention import read_back_pieces

    assert read_back_pieces([3, 4, 3], 10) == [(0, 3)] and read_back_pieces([3, 4, 4], 10) == [(0, 2), (2, 3)]
    assert read_back_pieces([30, 4, 4, 11, 1], 10) == [(0, 1), (1, 3), (3, 4), (4, 5)]  # a longer request has its own
    assert read_back_pieces([4, 4, 4, 4], 12) == [(0, 2), (2, 4)]  # and the pieces are about equal
    assert read_back_pieces([7], 0) == [(0, 1)] and read_back_pieces([1, 1], 0) == [(0, 1), (1, 2)]


@pytest.mark.parametrize("kv_dtype", ["auto", "int4"])
@pytest.mark.parametrize("row,length,copied", [(64, 20, 32), (64, 0, 0), (64, 64, 64), (7, 3, 7), (31, 5, 31), (8192, 5000, 5024), (8192, 100, 112)])
def test_a_contiguous_fork_copies_no_more_than_its_length_asks_for(row, length, copied, kv_dtype):
    """Rows are copied in equal parts (16 positions or more, 256 parts at most), not whole."""
    from astrai_b200.inference.cache import PagePool, TaskCacheManager

    pool = PagePool(2, 1, 32, 3, row, "cpu", torch.float32, kv_dtype=kv_dtype)
    tc = TaskCacheManager(pool)
    assert tc.task_alloc("a", list(range(length)))
    for t in pool.storage.pools():
        t.copy_(torch.randint(1, 100, t.shape))
    before = [t.clone() for t in pool.storage.pools()]
    assert tc.task_fork("a", "b")
    a, b = tc.state("a").req_idx * row, tc.state("b").req_idx * row
    for t, old in zip(pool.storage.pools(), before):
        assert torch.equal(t[:, b:b + copied], old[:, a:a + copied])
        t[:, b:b + copied] = old[:, b:b + copied]
        assert torch.equal(t, old)  # nothing else has changed


def test_shapes_that_do_not_fit_are_refused_on_the_cpu_too():
    from astrai_b200 import ops

    pools = _pools(16, 2, 32)
    q, table, rows, lens = torch.randn(3, 4, 32), torch.arange(12).int().view(3, 4), torch.arange(3).int(), torch.tensor([4, 2, 1])
    new = torch.randn(3, 2, 32).bfloat16()
    before = [t.clone() for t in pools]
    for bad in (dict(seq_lens=lens[:2]), dict(req_pool_indices=rows[:2]), dict(q=q[:2]), dict(q=q[0]), dict(req_to_token=table[0]),
                dict(k_new=new[:2], v_new=new[:2]), dict(out=torch.empty(2, 4, 32)), dict(seq_lens=lens[:, None])):
        with pytest.raises(ValueError, match="kv4_decode"):
            ops.kv4_decode(**{**dict(q=q, k_codes=pools[0], k_meta=pools[1], v_codes=pools[2], v_meta=pools[3], req_to_token=table,
                                     req_pool_indices=rows, seq_lens=lens), **bad})
    with pytest.raises(ValueError, match="kv4_gather"):
        ops.kv4_gather(*pools, rows[:, None])
    assert all(torch.equal(t, b) for t, b in zip(pools, before))


def test_a_captured_step_is_told_the_longest_length_a_request_can_have(model):
    """A graph outlives the lengths of its capture: a back end that sizes its work by ``max_len`` gets a bound that holds."""
    sched = _scheduler(model)
    ex = sched._executor
    assert ex.task_cache.task_alloc("a", [1, 2, 3])
    kv = ex.task_cache.bind(["a"], ex.workspace)
    assert kv.max_len == 3 and ex._padded(kv, 1, 2).max_len == 48


def test_a_replica_cut_over_two_ranks_serves_forks_over_a_four_bit_cache(tmp_path):
    import json
    import os

    from helpers import launch_ranks

    out, root = str(tmp_path / "res"), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code, log = launch_ranks(2, os.path.join(root, "tests", "workers", "tp_kv4.py"), ["--out", out], 29786, cwd=root)
    assert code == 0, log
    a, b = (json.load(open(f"{out}.{r}")) for r in range(2))
    assert a["pool"] == b["pool"] == [[1, 16], [1, 1, 2]] * 2  # one of the two kv heads of 32 numbers each
    assert a["greedy"] == b["greedy"] == a["alone"] and all(len(g) == 8 for g in a["greedy"])
    assert a["sampled"] == b["sampled"] and a["sampled"][0] != a["sampled"][1]
    assert a["chunked"] == b["chunked"] == [g for i, g in enumerate(a["alone"]) if i % 3 < 2]
