"""What is measured of the operators of the 4-bit KV cache: storing rows, reading them back, decode attention, prefill
attention and the copying of pages.

The cache keeps a key or value row of ``D`` numbers per token and head in groups of 32.  A group holds a step ``s`` and a
middle ``m`` (bf16 each) and 32 codes ``c`` of four bits; a number reads back as ``m + s * (c - 8)``.  With ``lo`` and
``hi`` the group's least and greatest number: ``s = bf16((hi - lo) / 15)``, ``m = bf16(lo + 8 s)`` and
``c = clamp(round((x - m) / s), -8, 7) + 8`` (``c = 8`` where ``s`` is 0).

Codes are held in the order in which the attention kernel's lanes read them, two to a byte (the lower half first): keys as
``[quarter of a group][group][8]``, four groups at a time, values as ``[eighth of a group][group][4]``.
"""

import math
import random

import torch

own = False

PAGE = 16  # tokens of a page


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # four chats that have just begun, on the smallest model: latency is all there is
        dict(name="decode: 4 short, 4/2 x 64", op="decode", batch=4, shortest=1, longest=33, heads=4, kv_heads=2, dim=64, store=False),
        # a full serving batch of mixed lengths on the 1B model, the step's own rows stored in the same call
        dict(name="decode: 128 mixed, 16/4 x 128", op="decode", batch=128, shortest=16, longest=4608, heads=16, kv_heads=4, dim=128, store=True),
        # one request over a book-length prompt on the 8B model: few rows, a long axis
        dict(name="decode: 1 long, 32/8 x 128", op="decode", batch=1, shortest=65521, longest=65521, heads=32, kv_heads=8, dim=128, store=False),
        # the reference's default model (24 heads of 64 over 4), a medium batch of long chats
        dict(name="decode: 32 long, 24/4 x 64", op="decode", batch=32, shortest=2049, longest=8191, heads=24, kv_heads=4, dim=64, store=False),
        # the rows of one decode step of 16 requests
        dict(name="store: 16 rows, 4 x 128", op="store", tokens=16, kv_heads=4, dim=128),
        # a whole prefill chunk of the 8B model
        dict(name="store: 8192 rows, 8 x 128", op="store", tokens=8192, kv_heads=8, dim=128),
        # the keys and values of a short ragged prefill batch
        dict(name="read: 237 rows, 4 x 64", op="read", tokens=237, kv_heads=4, dim=64),
        # the cached history that a prefill chunk at the end of long prompts attends to
        dict(name="read: 131072 rows, 8 x 128", op="read", tokens=131072, kv_heads=8, dim=128),
        # new prompts of odd lengths, nothing cached
        dict(name="prefill: 6 fresh, 16/4 x 128", op="prefill", batch=6, shortest=41, longest=1111, cached=0, heads=16, kv_heads=4, dim=128),
        # a chunk at the end of a long prompt (chunked prefill)
        dict(name="prefill: 1 chunk, 32/8 x 128", op="prefill", batch=1, shortest=1024, longest=1024, cached=15331, heads=32, kv_heads=8, dim=128),
        # one sequence is forked: the page that it shares only in part is copied, in every layer
        dict(name="pages: 1, 24 layers 4 x 128", op="pages", pages=1, pool=64, layers=24, kv_heads=4, dim=128),
        # a whole prefix is copied for several continuations
        dict(name="pages: 192, 32 layers 8 x 128", op="pages", pages=192, pool=512, layers=32, kv_heads=8, dim=128),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "store", "read", "prefill", "pages"])
    dim = rng.choice([32, 64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 6, 7, 8])
    if op == "decode":
        batch = _spread(rng, 1, 128)
        longest = _spread(rng, 1, min(65536, max(1, (65536 * 1024) // (batch * kv_heads * dim))))
        shortest = _spread(rng, 1, longest)
        return dict(op=op, batch=batch, shortest=shortest, longest=longest, heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    store=rng.random() < 0.5)
    if op in ("store", "read"):
        return dict(op=op, tokens=_spread(rng, 1, (2 ** 23 if op == "store" else 2 ** 27) // (kv_heads * dim)), kv_heads=kv_heads, dim=dim)
    if op == "prefill":
        dim = rng.choice([64, 128])
        batch = _spread(rng, 1, 6)
        longest = _spread(rng, 1, 1024 // batch)
        return dict(op=op, batch=batch, shortest=_spread(rng, 1, longest), longest=longest,
                    cached=rng.choice([0, _spread(rng, 1, 4096)]), heads=kv_heads * group, kv_heads=kv_heads, dim=dim)
    return dict(op=op, pages=_spread(rng, 1, 128), pool=rng.randint(260, 400), layers=rng.randint(1, 32), kv_heads=kv_heads,
                dim=rng.choice([32, 64, 128]))


def _lens(case):
    """The lengths of a batch: fixed by the case, spread evenly over the logarithm, longest first."""
    rng = random.Random("%d %d %d" % (case["batch"], case["shortest"], case["longest"]))
    lens = [_spread(rng, case["shortest"], case["longest"]) for _ in range(case["batch"])]
    lens[0] = case["longest"]
    return lens


def work(case):
    row = case["kv_heads"] * case["dim"]
    packed = 2 * row * 5 // 8  # codes and steps / middles of a token's key and value rows
    if case["op"] == "decode":
        n, b = sum(_lens(case)), case["batch"]
        fresh = b * (4 * row + packed + 4 * row) if case["store"] else 0
        return {"bytes": n * (packed + 4) + 4 * b * case["heads"] * case["dim"] + fresh, "flops": 4 * n * case["heads"] * case["dim"]}
    if case["op"] == "store":  # rows in, codes out; the rows are read back
        return {"bytes": case["tokens"] * (4 * row + 2 * packed + 4 * row), "flops": case["tokens"] * 2 * row * 8}
    if case["op"] == "read":
        return {"bytes": case["tokens"] * (packed + 4 * row + 4), "flops": case["tokens"] * 2 * row * 2}
    if case["op"] == "prefill":
        new = _lens(case)
        total, cached = sum(new), case["cached"]
        pairs = sum(n * cached + n * (n + 1) // 2 for n in new)
        keys = total + cached * len(new)
        return {"bytes": total * (4 * row + packed + 4 * row) + keys * packed + 4 * total * case["heads"] * case["dim"],
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    return {"bytes": 2 * case["pages"] * PAGE * case["layers"] * packed, "flops": 0}


# ----------------------------------------------------------------------------------------------------- the plain forms
def _pack(c, keys):
    """Codes ``[..., D]`` in the order of the row -> bytes ``[..., D / 2]`` in the order of the cache."""
    lead, d = c.shape[:-1], c.shape[-1]
    g = d // 32
    if keys:
        q = min(g, 4)
        c = c.reshape(*lead, g // q, q, 4, 8).transpose(-2, -3)
    else:
        c = c.reshape(*lead, g, 8, 4).transpose(-2, -3)
    c = c.reshape(*lead, d // 2, 2)
    return (c[..., 0] | (c[..., 1] << 4)).to(torch.uint8)


def _unpack(b, keys):
    """Bytes ``[..., D / 2]`` -> codes ``[..., D]`` (the reverse of :func:`_pack`)."""
    lead, d = b.shape[:-1], b.shape[-1] * 2
    g = d // 32
    c = torch.stack((b & 15, b >> 4), dim=-1)
    if keys:
        q = min(g, 4)
        return c.reshape(*lead, g // q, 4, q, 8).transpose(-2, -3).reshape(*lead, d)
    return c.reshape(*lead, 8, g, 4).transpose(-2, -3).reshape(*lead, d)


def _quantise(x, keys):
    """bf16 rows ``[..., D]`` -> codes ``[..., D / 2]`` and ``(m, s)`` ``[..., D / 32, 2]``."""
    x = x.float().unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi - lo) / 15).to(torch.bfloat16)
    s32 = s.float()
    m = (lo + 8 * s32).to(torch.bfloat16)
    c = torch.where(s32 > 0, ((x - m.float()) / s32).round().clamp(-8, 7) + 8, torch.full_like(x, 8.0))
    return _pack(c.to(torch.uint8).flatten(-2), keys), torch.cat((m, s), dim=-1)


def _values(codes, meta, keys):
    """What the cache stands for, in 32 bits."""
    c = _unpack(codes, keys).float().unflatten(-1, (-1, 32)) - 8
    return (meta[..., :1].float() + meta[..., 1:].float() * c).flatten(-2)


def _plain_store(st):
    for x, codes, meta, keys in ((st["k"], st["k_codes"], st["k_meta"], True), (st["v"], st["v_codes"], st["v_meta"], False)):
        c, ms = _quantise(x, keys)
        codes[st["loc"]] = c
        meta[st["loc"]] = ms


def _plain_read(st, loc):
    return (_values(st["k_codes"][loc], st["k_meta"][loc], True).to(torch.bfloat16),
            _values(st["v_codes"][loc], st["v_meta"][loc], False).to(torch.bfloat16))


def _plain_attention(q, k, v, hidden):
    """``q [B, S, Hq, D]``, ``k / v [B, L, Hkv, D]`` in 32 bits; ``hidden [B, S, L]`` marks what is not attended to."""
    b, s, hq, d = q.shape
    hkv = k.shape[2]
    q = q.reshape(b, s, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    p = torch.matmul(q, k.permute(0, 2, 3, 1)) * d ** -0.5
    p = p.view(b, hkv, hq // hkv, s, -1).masked_fill_(hidden[:, None, None], -math.inf).view(b, hkv, (hq // hkv) * s, -1)
    p = (p - p.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3))
    return o.view(b, hkv, hq // hkv, s, d).permute(0, 3, 1, 2, 4).reshape(b, s, hq, d)


def _plain_decode(st):
    if st["k"] is not None:
        _plain_store(st)
    longest = st["max_len"]
    slots = st["table"][st["rows"].long(), :longest].long()
    at = torch.arange(longest, device=slots.device)
    hidden = (at[None] >= st["lens"][:, None])
    k = _values(st["k_codes"][slots], st["k_meta"][slots], True)
    v = _values(st["v_codes"][slots], st["v_meta"][slots], False)
    return _plain_attention(st["q"].float()[:, None], k, v, hidden[:, None])[:, 0].to(torch.bfloat16)


def _plain_prefill(st):
    """Ragged queries at the end of their requests' keys: padded to the longest, all requests at once."""
    _plain_store(st)
    q_lens = st["qo_indptr"][1:] - st["qo_indptr"][:-1]
    kv_lens = st["lens"]
    b, sq, sk = q_lens.numel(), max(st["q_lens"]), st["max_len"]
    at_q = torch.arange(sq, device=q_lens.device)
    at_k = torch.arange(sk, device=q_lens.device)
    k, v = _plain_read(st, st["table"][st["rows"].long(), :sk].long())
    token = (st["qo_indptr"][:-1, None] + at_q).clamp(max=st["q"].shape[0] - 1).long()
    last = (kv_lens - q_lens)[:, None] + at_q  # the last key that a query sees
    hidden = at_k[None, None] > last[:, :, None]
    out = _plain_attention(st["q"][token].float(), k.float(), v.float(), hidden)
    return out[at_q[None] < q_lens[:, None]].to(torch.bfloat16)


def _plain_pages(st):
    page = torch.arange(PAGE)
    src = (torch.tensor(st["src"])[:, None] * PAGE + page).reshape(-1).to(st["pools"][0].device)
    dst = (torch.tensor(st["dst"])[:, None] * PAGE + page).reshape(-1).to(st["pools"][0].device)
    for pool in st["pools"]:
        pool[:, dst] = pool[:, src]


# ------------------------------------------------------------------------------------------------------------ the state
def _rows(gen, tokens, kv_heads, dim, offset):
    """Key or value rows as a projection gives them: channels of unequal width, a few of them far from zero."""
    wide = torch.exp(0.5 * torch.randn(kv_heads, dim, generator=gen, device="cuda"))
    middle = offset * torch.randn(kv_heads, dim, generator=gen, device="cuda")
    return (torch.randn(tokens, kv_heads, dim, generator=gen, device="cuda") * wide + middle).to(torch.bfloat16)


def _cache(gen, slots, kv_heads, dim):
    """Codes and (m, s) of ``slots`` filled rows, keys and values; made a piece at a time to bound the memory it takes."""
    made = {"k": ([], []), "v": ([], [])}
    piece = max(1, 2 ** 25 // (kv_heads * dim))
    for start in range(0, slots, piece):
        n = min(piece, slots - start)
        for name, offset in (("k", 1.0), ("v", 0.2)):
            c, ms = _quantise(_rows(gen, n, kv_heads, dim, offset), name == "k")
            made[name][0].append(c)
            made[name][1].append(ms)
    return {"k_codes": torch.cat(made["k"][0]), "k_meta": torch.cat(made["k"][1]),
            "v_codes": torch.cat(made["v"][0]), "v_meta": torch.cat(made["v"][1])}


def _table(gen, lens, width):
    """Pages of 16 tokens, handed out in any order: ``table[r, t]`` is the slot of token ``t`` of row ``r``."""
    per = [-(-n // PAGE) for n in lens]
    order = torch.randperm(sum(per), generator=gen, device="cuda")
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    inside = torch.arange(PAGE, device="cuda")
    start = 0
    for row, (n, p) in enumerate(zip(lens, per)):
        table[row, :n] = (order[start:start + p, None] * PAGE + inside).reshape(-1)[:n].int()
        start += p
    return table, sum(per) * PAGE


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, kv_heads, dim = case["op"], case["kv_heads"], case["dim"]
    if op == "pages":
        shape = (case["layers"], case["pool"] * PAGE, kv_heads)
        order = torch.randperm(case["pool"], generator=gen, device="cuda").tolist()
        codes = [torch.randint(0, 256, (*shape, dim // 2), generator=gen, device="cuda", dtype=torch.uint8) for _ in range(2)]
        meta = [torch.randn(*shape, dim // 32, 2, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2)]
        return {"op": op, "pools": [codes[0], meta[0], codes[1], meta[1]], "src": order[:case["pages"]],
                "dst": order[case["pages"]:2 * case["pages"]]}
    if op in ("store", "read"):
        n = case["tokens"]
        slots = -(-n // PAGE) * PAGE * 2
        loc = torch.randperm(slots, generator=gen, device="cuda")[:n]
        st = {"op": op, "loc": loc, **_cache(gen, slots, kv_heads, dim)}
        if op == "store":
            st["k"], st["v"] = _rows(gen, n, kv_heads, dim, 1.0), _rows(gen, n, kv_heads, dim, 0.2)
        return st
    new = _lens(case)
    cached = case["cached"] if op == "prefill" else 0
    lens = [n + cached for n in new]
    width = -(-max(lens) // PAGE) * PAGE
    table, slots = _table(gen, lens, width)
    st = {"op": op, "table": table, "rows": torch.arange(len(lens), dtype=torch.int32, device="cuda"), "max_len": max(lens),
          "lens": torch.tensor(lens, device="cuda"), "kv_lens": lens, "k": None, "v": None, **_cache(gen, slots, kv_heads, dim)}
    tokens = len(lens) if op == "decode" else sum(new)
    st["q"] = torch.randn(tokens, case["heads"], dim, generator=gen, device="cuda").to(torch.bfloat16)
    if op == "prefill" or case["store"]:
        st["k"], st["v"] = _rows(gen, tokens, kv_heads, dim, 1.0), _rows(gen, tokens, kv_heads, dim, 0.2)
    if op == "decode":
        st["loc"] = table[st["rows"].long(), st["lens"] - 1].long()
        b, splits = len(lens), 32  # the scratch that a serving workspace keeps
        st["workspace"] = (torch.zeros(b, case["heads"], splits, dim, device="cuda"), torch.zeros(b, case["heads"], splits, 2, device="cuda"),
                           torch.zeros(b * kv_heads, dtype=torch.int32, device="cuda"))
        return st
    st["q_lens"] = new
    st["loc"] = torch.cat([table[i, cached:n] for i, n in enumerate(lens)]).long()
    st["all_loc"] = torch.cat([table[i, :n] for i, n in enumerate(lens)]).long()
    st["qo_indptr"] = torch.tensor([0] + new, device="cuda").cumsum(0).int()
    st["kv_indptr"] = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    return st


# ----------------------------------------------------------------------------------------------------------------- run
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    op = st["op"]
    if op == "pages":
        _plain_pages(st)
        return st["pools"]
    if op == "store":
        _plain_store(st)
        return _plain_read(st, st["loc"])
    if op == "read":
        return _plain_read(st, st["loc"])
    out = _plain_decode(st) if op == "decode" else _plain_prefill(st)
    return (out, *_plain_read(st, st["loc"])) if st["k"] is not None else (out,)


def _run_own(st):
    from astrai_b200 import ops

    op = st["op"]
    if op == "pages":
        ops.copy_pages_(st["pools"], st["src"], st["dst"], PAGE)
        return st["pools"]
    pools = (st["k_codes"], st["k_meta"], st["v_codes"], st["v_meta"])
    if op == "store":
        ops.kv4_append_(st["k"], st["v"], *pools, st["loc"])
        return ops.kv4_gather(*pools, st["loc"])
    if op == "read":
        return ops.kv4_gather(*pools, st["loc"])
    if op == "decode":
        out = ops.kv4_decode(st["q"], *pools, st["table"], st["rows"], st["lens"], k_new=st["k"], v_new=st["v"],
                             max_len=st["max_len"], workspace=st["workspace"])
    else:
        cache = ops.KVCache(k_buffer=pools[0][None], k_meta=pools[1][None], v_buffer=pools[2][None], v_meta=pools[3][None],
                            req_to_token=st["table"], req_pool_indices=st["rows"], seq_lens=st["lens"], out_cache_loc=st["loc"],
                            max_len=st["max_len"], kv_indptr=st["kv_indptr"], qo_indptr=st["qo_indptr"], q_lens=st["q_lens"],
                            kv_lens=st["kv_lens"], kv_gather_loc=st["all_loc"], page_size=PAGE)
        out = ops.attention(st["q"], st["k"], st["v"], cache, 0, None, True, "prefill")
    return (out, *ops.kv4_gather(*pools, st["loc"])) if st["k"] is not None else (out,)


# --------------------------------------------------------------------------------------------------------------- exact
def _exact_codes(rows):
    """From the definition, a group at a time: ``(m, s, c - 8)`` of rows ``[n, heads, D]`` as ``[n, heads, D / 32, ...]``, 64 bits."""
    x = rows.double().reshape(*rows.shape[:2], -1, 32)
    low, high = torch.aminmax(x, dim=3)
    step = ((high - low) / 15.0).to(torch.bfloat16).double()
    mid = (low + 8.0 * step).to(torch.bfloat16).double()
    safe = torch.where(step == 0.0, torch.ones_like(step), step)
    c = torch.round((x - mid[..., None]) / safe[..., None])
    c = torch.minimum(torch.maximum(c, torch.full_like(c, -8.0)), torch.full_like(c, 7.0))
    return mid, step, torch.where(step[..., None] == 0.0, torch.zeros_like(c), c)


def _exact_rows(rows):
    mid, step, c = _exact_codes(rows)
    return (mid[..., None] + step[..., None] * c).reshape(rows.shape)


def _place(dim, keys, device):
    """``place[i]``: where among a row's nibbles number ``i`` of the row is held."""
    i = torch.arange(dim, device=device)
    group, inside = i // 32, i % 32
    groups = dim // 32
    if not keys:
        return (inside // 4) * (groups * 4) + group * 4 + inside % 4
    four = min(groups, 4)
    return (group // four) * (32 * four) + (inside // 8) * (8 * four) + (group % four) * 8 + inside % 8


def _exact_read(codes, meta, keys):
    """Rows of the cache ``[n, heads, D / 2]`` in 64 bits, nibble by nibble."""
    n, heads, half = codes.shape
    place = _place(2 * half, keys, codes.device)
    byte = codes[..., place // 2].int()
    nibble = torch.where((place % 2).bool(), byte // 16, byte % 16).double() - 8.0
    number = nibble.reshape(n, heads, -1, 32) * meta[..., 1].double()[..., None] + meta[..., 0].double()[..., None]
    return number.reshape(n, heads, 2 * half)


def _exact_softmax_attention(q, k, v, first):
    """``q [S, Hq, D]`` over ``k / v [L, Hkv, D]``; query ``i`` sees the keys up to ``first + i``."""
    group = q.shape[1] // k.shape[1]
    seen = torch.arange(k.shape[0], device=q.device)[None] <= first + torch.arange(q.shape[0], device=q.device)[:, None]
    heads = []
    for h in range(q.shape[1]):
        logit = (q[:, h] @ k[:, h // group].T) / math.sqrt(q.shape[2])
        weight = torch.softmax(torch.where(seen, logit, torch.full_like(logit, -math.inf)), dim=1)
        heads.append(weight @ v[:, h // group])
    return torch.stack(heads, dim=1)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "pages":
        at = torch.arange(case["pool"], device="cuda")
        at[torch.tensor(st["dst"], device="cuda")] = torch.tensor(st["src"], device="cuda")  # which page each one now equals
        return [p.unflatten(1, (-1, PAGE))[:, at].flatten(1, 2) for p in st["pools"]]
    if op == "store":
        return _exact_rows(st["k"]), _exact_rows(st["v"])
    if op == "read":
        return (_exact_read(st["k_codes"][st["loc"]], st["k_meta"][st["loc"]], True),
                _exact_read(st["v_codes"][st["loc"]], st["v_meta"][st["loc"]], False))
    fresh = (_exact_rows(st["k"]), _exact_rows(st["v"])) if st["k"] is not None else ()
    outs, start = [], 0
    for row, length in enumerate(st["kv_lens"]):
        count = 1 if op == "decode" else st["q_lens"][row]
        slots = st["table"][row, :length].long()
        k = _exact_read(st["k_codes"][slots], st["k_meta"][slots], True)
        v = _exact_read(st["v_codes"][slots], st["v_meta"][slots], False)
        if fresh:
            k[length - count:], v[length - count:] = fresh[0][start:start + count], fresh[1][start:start + count]
        if op == "prefill":  # a prompt's attention takes the rows as they are read back
            k, v = k.to(torch.bfloat16).double(), v.to(torch.bfloat16).double()
        outs.append(_exact_softmax_attention(st["q"][start:start + count].double(), k, v, length - count))
        start += count
    return (torch.cat(outs), *fresh)
