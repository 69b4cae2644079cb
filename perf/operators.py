"""Timing cases of the 4-bit paged KV cache operators.

Four operators over one cache format: storing rows (append and read back), attention, accumulating attention
weights per cached token, and evicting tokens by weight. ``run`` computes each one either in plain 32-bit torch
operations (``own`` false) or through ``kvbridge_b200`` (``own`` true), from the same device buffers.

Cache format: a row x of one token and KV head (``dim`` values) is held as codes 0..15 with
``lo = min x``, ``scale = (max x - min x) / 15``, ``value = lo + scale * code``; two dims to a byte (the even one
low). K bytes are ``[page, head, slot, dim / 2]``, V bytes ``[page, head, dim / 2, slot]``, the (scale, lo) pairs
float32 ``[page, head, slot, 2]``.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# Cases


def _store(name, **kw):
    return dict(op="store", name=name, tokens=1, kv_heads=8, dim=128, page=64, dtype="bf16", layout="scattered") | kw


def _attend(name, **kw):
    return dict(op="attend", name=name, batch=1, rows=1, q_heads=32, kv_heads=8, dim=128, page=64, low=1, high=4096,
                lens_seed=1, dtype="f16", softcap=0.0, slopes=False, window=0, prefix=0, positions=False) | kw


def _weigh(name, **kw):
    return _attend(name, **kw) | {"op": "weigh"}


def _evict(name, **kw):
    return dict(op="evict", name=name, batch=1, kv_heads=8, dim=128, page=64, low=1, high=4096, lens_seed=1, budget=1024,
                sinks=4, recent=128) | kw


def listed():
    return [
        # One decode step of 64 sequences: each writes one token to a page of its own (a launch's latency).
        _store("store step 64x1", tokens=64),
        # A whole long prompt of 65,536 tokens, written from inside a page on.
        _store("store prompt 64K", tokens=65536, layout="run"),
        # One decode row over a short context in fp32 (the smallest attention call).
        _attend("attend 1x4K f32", low=4096, high=4096, dtype="f32"),
        # One sequence of 65,536 tokens, 32/8 heads: the repository's headline decode shape.
        _attend("attend 1x64K", low=65536, high=65536),
        # Ragged batch of 32 sequences of 1K to 32K tokens.
        _attend("attend 32 ragged", batch=32, low=1024, high=32768, lens_seed=3, dtype="bf16"),
        # 64 sequences of 16K tokens, 64/8 heads, 16-token pages.
        _attend("attend 64x16K g8 p16", batch=64, q_heads=64, page=16, low=16384, high=16384, dtype="bf16"),
        # Eight query rows of one sequence (speculative decoding), 24/4 heads of 256 dims, prefix visible to all rows.
        _attend("attend 8 rows d256", rows=8, q_heads=24, kv_heads=4, dim=256, page=32, low=32768, high=32768, prefix=100),
        # A capped, windowed layer with attention sinks: 16 sequences, two rows each, lengths down to one token.
        _attend("attend capped window", batch=16, rows=2, low=1, high=20000, lens_seed=5, dtype="bf16", softcap=50.0,
                window=4096, prefix=16, slopes=True),
        # Accumulated weights of a short sequence with explicit positions (a cache that was compacted before).
        _weigh("weigh 1x5000 compacted", low=5000, high=5000, dtype="f16", slopes=True, positions=True),
        # Accumulated weights of a ragged batch, 64/8 heads.
        _weigh("weigh 32 ragged g8", batch=32, q_heads=64, low=1024, high=32768, lens_seed=7, dtype="bf16"),
        # Keeping 2,048 of 1,500 to 16K tokens of 16 sequences (some have fewer and keep all).
        _evict("evict 16x16K", batch=16, low=1500, high=16384, lens_seed=9, budget=2048),
        # Keeping an eighth of one sequence of 131,071 tokens, two KV heads, 32-token pages.
        _evict("evict 1x128K", kv_heads=2, page=32, low=131071, high=131071, budget=16384, recent=1000),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


#: KV values (tokens * KV heads * dim, K and V counted once) of the largest listed case.
MOST_VALUES = 64 * 16384 * 8 * 128


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "weigh", "evict"])
    kv_heads, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64])
    dtype = rng.choice(["f16", "bf16", "f32"])
    if op == "store":
        tokens = _log_int(rng, 1, 65536)
        case = _store("", tokens=tokens, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                      layout=rng.choice(["run", "scattered"]))
    else:
        batch = _log_int(rng, 1, 64)
        high = _log_int(rng, 1, max(1, min(131072, MOST_VALUES // (batch * kv_heads * dim))))
        low = max(1, high // rng.choice([1, 2, 8, high]))
        common = dict(batch=batch, kv_heads=kv_heads, dim=dim, page=page, low=low, high=high, lens_seed=rng.randrange(1000))
        if op == "evict":
            budget = max(1, high // rng.choice([1, 2, 3, 8]))
            recent = rng.randrange(0, budget // 2 + 1)
            case = _evict("", budget=budget, recent=recent, sinks=min(rng.choice([0, 1, 4]), budget - recent), **common)
        else:
            group = rng.choice([1, 2, 4, 5, 7, 8, 12, 16])
            # Columns times KV values no more than at 64 x 16K tokens with a group of 8.
            spare = 8 * MOST_VALUES // max(1, batch * high * kv_heads * dim)
            rows = rng.randint(1, max(1, min(8, 64 // group, spare // group)))
            case = (_attend if op == "attend" else _weigh)(
                "", rows=rows, q_heads=kv_heads * group, dtype=dtype, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                slopes=rng.random() < 0.3, window=rng.choice([0, 0, _log_int(rng, 1, 8192)]),
                prefix=rng.choice([0, 0, 1, 16, 100]), positions=rng.random() < 0.2, **common)
    del case["name"]
    return case


def _lengths(case):
    g = torch.Generator().manual_seed(case["lens_seed"])
    return [int(x) for x in torch.randint(case["low"], case["high"] + 1, (case["batch"],), generator=g)]


def _seen(case, length):
    """Cached tokens of one sequence that some query row of the call sees."""
    if not case["window"] or case["positions"]:
        return length  # a compacted cache has to be looked through
    first = max(0, length - case["rows"] - case["window"] + 1)
    return length - max(0, first - min(case["prefix"], length))


def work(case):
    heads, dim = case["kv_heads"], case["dim"]
    row = dim // 2 + 8  # bytes of a cached K (or V) row
    if case["op"] == "store":
        n = case["tokens"]
        dense = 2 * heads * dim * SIZES[case["dtype"]]
        return {"bytes": n * (2 * dense + 2 * 2 * heads * row + 2 * 8), "flops": n * heads * dim * 2 * 6}
    if case["op"] == "evict":
        lens = _lengths(case)
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": heads * (4 * sum(lens) + 2 * kept * (2 * row + 4) + kept * (4 + 4 + 4)), "flops": heads * sum(lens)}
    seen = sum(_seen(case, n) for n in _lengths(case))
    queries = case["batch"] * case["rows"] * case["q_heads"]
    size = SIZES[case["dtype"]]
    if case["op"] == "attend":
        extra = seen * heads * 4 if case["positions"] else 0
        return {"bytes": seen * heads * 2 * row + queries * (2 * dim * size + 4) + extra,
                "flops": 4 * seen * case["rows"] * case["q_heads"] * dim}
    extra = seen * heads * 4 if case["positions"] else 0
    return {"bytes": seen * heads * (row + 8) + queries * (dim * size + 4) + extra,
            "flops": 2 * seen * case["rows"] * case["q_heads"] * dim}


# ---------------------------------------------------------------------------
# Inputs


def _pack(x):
    """Codes (two to a byte along the last axis) and (scale, lo) of float rows x."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = (high - low) / 15
    code = ((x - low) / torch.where(scale > 0, scale, torch.ones_like(scale))).round().clamp(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([scale, low], -1)


def _unpack(code, params):
    """The values (float32) that packed rows stand for."""
    value = torch.stack([code & 15, code >> 4], -1).flatten(-2).float()
    return params[..., 1:] + params[..., :1] * value


def _cache(case, pages, g):
    """A pool of `pages` filled pages: keys with per-channel offsets and some large rows, values around zero."""
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    k = torch.empty((pages, heads, page, dim // 2), dtype=torch.uint8, device=DEVICE)
    v = torch.empty((pages, heads, dim // 2, page), dtype=torch.uint8, device=DEVICE)
    kp = torch.empty((pages, heads, page, 2), device=DEVICE)
    vp = torch.empty((pages, heads, page, 2), device=DEVICE)
    offset = torch.randn((heads, 1, dim), generator=g, device=DEVICE)
    chunk = max(1, (1 << 26) // (heads * page * dim))
    for p in range(0, pages, chunk):
        n = min(chunk, pages - p)
        x = torch.randn((n, heads, page, dim), generator=g, device=DEVICE) + offset
        k[p:p + n], kp[p:p + n] = _pack(x)
        x = torch.randn((n, heads, page, dim), generator=g, device=DEVICE)
        x *= 1 + 9 * (torch.rand((n, heads, page, 1), generator=g, device=DEVICE) < 0.01)
        code, vp[p:p + n] = _pack(x)
        v[p:p + n] = code.transpose(-1, -2)
    return k, v, kp, vp


def _tables(case, g, spare=0):
    """Sequence lengths, the block table over a shuffled pool, and the number of pages."""
    lens = _lengths(case)
    each = [-(-n // case["page"]) for n in lens]
    order = torch.randperm(sum(each), generator=g, device=DEVICE).to(torch.int32)
    width = max(each)
    at = torch.arange(width, device=DEVICE)
    starts = torch.tensor([sum(each[:i]) for i in range(len(each))], device=DEVICE)
    counts = torch.tensor(each, device=DEVICE)
    table = torch.where(at < counts[:, None], order[(starts[:, None] + at).clamp(max=len(order) - 1)],
                        torch.zeros((), dtype=torch.int32, device=DEVICE)).contiguous()
    return torch.tensor(lens, dtype=torch.int32, device=DEVICE), table, sum(each)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {"case": case}
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "store":
        n, kind = case["tokens"], TYPES[case["dtype"]]
        # The pool holds other sequences' pages too; a run of tokens starts inside a page.
        pages = n + 2 if case["layout"] == "scattered" and n <= 1024 else -(-n // page) + 3
        order = torch.randperm(pages, generator=g, device=DEVICE)
        if case["layout"] == "run":
            at = torch.arange(n, device=DEVICE) + page // 2 + 1
            s["slots"] = order[at // page] * page + at % page
        elif n <= 1024:
            s["slots"] = order[:n] * page + torch.randint(0, page, (n,), generator=g, device=DEVICE)
        else:
            s["slots"] = torch.randperm(pages * page, generator=g, device=DEVICE)[:n]
        # K and V are columns of one projection's output.
        rows = torch.randn((n, 3 * heads * dim), generator=g, device=DEVICE)
        rows[:, ::7] += 2
        rows = rows.to(kind)
        s["k_new"] = rows[:, heads * dim:2 * heads * dim].unflatten(1, (heads, dim))
        s["v_new"] = rows[:, 2 * heads * dim:].unflatten(1, (heads, dim))
        s["k"] = torch.zeros((pages, heads, page, dim // 2), dtype=torch.uint8, device=DEVICE)
        s["v"] = torch.zeros((pages, heads, dim // 2, page), dtype=torch.uint8, device=DEVICE)
        s["k_params"] = torch.zeros((pages, heads, page, 2), device=DEVICE)
        s["v_params"] = torch.zeros((pages, heads, page, 2), device=DEVICE)
        s["k_out"] = torch.empty((n, heads, dim), dtype=kind, device=DEVICE)
        s["v_out"] = torch.empty((n, heads, dim), dtype=kind, device=DEVICE)
        return s
    s["lens"], s["table"], used = _tables(case, g)
    batch = case["batch"]
    if case["op"] == "evict":
        budget = case["budget"]
        each = -(-budget // page)
        s["k"], s["v"], s["k_params"], s["v_params"] = _cache(case, used + batch * each, g)
        s["new_table"] = torch.arange(used, used + batch * each, dtype=torch.int32, device=DEVICE).view(batch, each)
        s["first_new"] = used
        s["positions"] = torch.randint(0, 1 << 20, s["k_params"].shape[:-1], generator=g, device=DEVICE, dtype=torch.int32)
        # Accumulated weights spread over orders of magnitude; tokens that nothing looked at share the value zero.
        w = torch.randn((batch, heads, case["high"]), generator=g, device=DEVICE)
        s["weights"] = torch.where(w < -1.5, 0.0, torch.exp(2 * w))
        s["keep"] = torch.zeros((batch, heads, budget), dtype=torch.int32, device=DEVICE)
        s["new_lens"] = torch.zeros((batch,), dtype=torch.int32, device=DEVICE)
        s["new_weights"] = torch.zeros((batch, heads, budget), device=DEVICE)
        return s
    s["k"], s["v"], s["k_params"], s["v_params"] = _cache(case, used, g)
    rows, q_heads, kind = case["rows"], case["q_heads"], TYPES[case["dtype"]]
    # Queries are columns of one projection's output.
    x = torch.randn((batch, rows, (q_heads + 2 * heads) * dim), generator=g, device=DEVICE) * 1.5
    s["q"] = x.to(kind)[..., :q_heads * dim].unflatten(2, (q_heads, dim))
    s["scale"] = 1 / math.sqrt(dim)
    s["slopes"] = None
    if case["slopes"]:
        s["slopes"] = torch.exp2(-8 * (torch.arange(q_heads, device=DEVICE) + 1) / q_heads)
    s["prefix"] = None
    if case["prefix"]:
        s["prefix"] = torch.full((batch,), case["prefix"], dtype=torch.int32, device=DEVICE)
    s["positions"] = s["q_positions"] = None
    if case["positions"]:
        # About one token in three was kept by each head; the rows are the next tokens of the sequence.
        steps = torch.randint(1, 6, (batch, heads, case["high"]), generator=g, device=DEVICE)
        at = steps.cumsum(-1).to(torch.int32)
        s["positions"] = torch.zeros(s["k_params"].shape[:-1], dtype=torch.int32, device=DEVICE)
        width = s["table"].shape[1] * page
        spread = torch.zeros((batch, heads, width), dtype=torch.int32, device=DEVICE)
        spread[..., :case["high"]] = at
        spread = spread.unflatten(2, (-1, page)).transpose(1, 2)
        real = torch.arange(s["table"].shape[1], device=DEVICE) * page < s["lens"][:, None]
        s["positions"][s["table"][real].long()] = spread[real]
        last = at.gather(-1, (s["lens"].long() - 1)[:, None, None].expand(-1, heads, 1)).amax(1)
        s["q_positions"] = (last + 1 + torch.arange(rows, device=DEVICE)).to(torch.int32).contiguous()
    if case["op"] == "attend":
        s["out"] = torch.empty((batch, rows, q_heads, dim), dtype=kind, device=DEVICE)
        s["lse"] = torch.empty((batch, rows, q_heads), device=DEVICE)
    else:
        # The log-sum-exp of each query row, as the attention call before it returns it.
        s["lse"] = _row_lse(s)
        # What a few steps left: about a step's share of a token, each.
        share = rows * q_heads / heads / case["high"]
        s["weights"] = torch.rand((batch, heads, case["high"]), generator=g, device=DEVICE) * share
    return s


# ---------------------------------------------------------------------------
# Plain forms, in 32 bits


def _plain_store(s):
    slots, page = s["slots"], s["case"]["page"]
    at, slot = slots // page, slots % page
    code, s["k_params"][at, :, slot] = _pack(s["k_new"].float())
    s["k"][at, :, slot] = code
    code, s["v_params"][at, :, slot] = _pack(s["v_new"].float())
    s["v"][at, :, :, slot] = code
    kind = s["k_new"].dtype
    return {"k": _unpack(s["k"][at, :, slot], s["k_params"][at, :, slot]).to(kind),
            "v": _unpack(s["v"][at, :, :, slot], s["v_params"][at, :, slot]).to(kind)}


def _keys(s):
    table = s["table"].long()
    return _unpack(s["k"][table], s["k_params"][table]).transpose(1, 2).flatten(2, 3)  # [batch, head, token, dim]


def _values(s):
    table = s["table"].long()
    return _unpack(s["v"][table].transpose(-1, -2), s["v_params"][table]).transpose(1, 2).flatten(2, 3)


def _scores(s):
    """Scores [batch, KV head, row, head of the group, token], masked ones at -inf."""
    case, q = s["case"], s["q"].float()
    rows, heads = case["rows"], case["kv_heads"]
    k = _keys(s)
    q = q.unflatten(2, (heads, -1)).transpose(1, 2)  # [batch, KV head, row, group, dim]
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (rows, -1)) * s["scale"]
    at = torch.arange(k.shape[2], device=q.device, dtype=torch.int32)
    lens = s["lens"][:, None, None, None]
    if s["positions"] is None:
        pk = at[None, None, None, :]
        pq = (s["lens"][:, None] - rows + torch.arange(rows, device=q.device, dtype=torch.int32))[:, None, :, None]
    else:
        pk = s["positions"][s["table"].long()].transpose(1, 2).flatten(2, 3)[:, :, None, :]
        pq = s["q_positions"][:, None, :, None]
    away = pq - pk
    sees = away >= 0
    if case["window"]:
        sees = sees & (away < case["window"])
    if s["prefix"] is not None:
        sees = sees | (pk < s["prefix"][:, None, None, None])
    sees = sees & (at < lens)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].view(heads, 1, -1, 1) * away.abs().unsqueeze(3)
    return x.masked_fill(~sees.unsqueeze(3), -math.inf)


def _row_lse(s):
    x = _scores(s)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    return (top + (x - top).exp().sum(-1, keepdim=True).log()).squeeze(-1).transpose(1, 2).flatten(2, 3).contiguous()


def _plain_attend(s):
    x = _scores(s)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (x - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), _values(s)).unflatten(2, (s["case"]["rows"], -1))
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log()).squeeze(-1)
    return {"out": out.transpose(1, 2).flatten(2, 3).to(s["q"].dtype), "lse": lse.transpose(1, 2).flatten(2, 3)}


def _plain_weigh(s):
    x = _scores(s)
    lse = s["lse"].unflatten(2, (s["case"]["kv_heads"], -1)).transpose(1, 2).unsqueeze(-1)
    p = torch.where(x == -math.inf, 0.0, (x - lse).exp())
    n = min(p.shape[-1], s["weights"].shape[-1])
    s["weights"][..., :n] += p.sum((2, 3))[..., :n]
    return {"weights": s["weights"]}


def _plain_evict(s):
    case = s["case"]
    budget, page, heads = case["budget"], case["page"], case["kv_heads"]
    weights, lens = s["weights"], s["lens"][:, None, None]
    at = torch.arange(weights.shape[-1], device=weights.device)
    always = (at < case["sinks"]) | (at >= lens - case["recent"])
    rank = torch.where(always, math.inf, weights)
    rank = torch.where(at < lens, rank, -math.inf)
    order = rank.argsort(dim=-1, descending=True, stable=True)[..., :budget]
    if order.shape[-1] < budget:
        order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]), value=weights.shape[-1])
    taken = torch.arange(budget, device=weights.device) < lens
    keep = torch.where(taken, order, weights.shape[-1]).sort(-1).values
    index = torch.where(taken, keep, 0)
    new_lens = s["lens"].clamp(max=budget)
    # Copy the kept tokens, head by head, into the new pages.
    head = torch.arange(heads, device=weights.device)[:, None]
    row = torch.arange(case["batch"], device=weights.device)[:, None, None]
    source, slot = s["table"].long()[row, index // page], index % page
    to = torch.arange(budget, device=weights.device)
    target = s["new_table"].long()[row, to // page].expand(-1, heads, -1)
    moved = taken.expand_as(index)
    source, slot, head, target, to = (t.expand_as(index)[moved] for t in (source, slot, head, target, to % page))
    s["k"][target, head, to] = s["k"][source, head, slot]
    s["v"][target, head, :, to] = s["v"][source, head, :, slot]
    for name in ("k_params", "v_params", "positions"):
        s[name][target, head, to] = s[name][source, head, slot]
    new_weights = torch.where(taken, weights.gather(-1, index), 0.0)
    return _evicted(s, index.to(torch.int32), new_lens, new_weights)


def _evicted(s, keep, new_lens, new_weights):
    # The new pages come back as stored: a moved token's bytes are those of the old one, so nothing may differ.
    new = {name: s[name][s["first_new"]:] for name in ("k", "v", "k_params", "v_params", "positions")}
    return new | {"keep": keep, "lens": new_lens, "weights": new_weights}


# ---------------------------------------------------------------------------
# The framework's operators


def _handles(s):
    """The pool, query and workspace objects that a serving program makes once for its buffers."""
    import kvbridge_b200 as kvb

    case = s["case"]
    s["pool"] = kvb.Kv4Pool(s["k"], s["v"], s["k_params"], s["v_params"], positions=s.get("positions"))
    if case["op"] == "store":
        s["new_rows"] = kvb.Kv4Rows(s["k_new"], s["v_new"], s["slots"])
        s["read_rows"] = kvb.Kv4Rows(s["k_out"], s["v_out"], s["slots"])
    elif case["op"] == "evict":
        s["plan"] = kvb.EvictPlan(s["weights"], s["lens"], s["table"], budget=case["budget"], sinks=case["sinks"],
                                  recent=case["recent"])
    else:
        s["query"] = kvb.Kv4Query(s["q"], s["lens"], s["table"], max_tokens=case["high"], kv_heads=case["kv_heads"],
                                  scale=s["scale"], softcap=case["softcap"], slopes=s["slopes"], window=case["window"],
                                  prefix_lens=s["prefix"], q_positions=s["q_positions"])
        if case["op"] == "attend":
            size = kvb.attention_kv4_workspace_bytes(s["pool"], s["query"])
            s["workspace"] = torch.empty(size, dtype=torch.uint8, device=DEVICE)
    return kvb


def _own_pass(s):
    kvb = s.get("library")
    if kvb is None:
        kvb = s["library"] = _handles(s)
    op = s["case"]["op"]
    if op == "store":
        kvb.append_kv4(s["pool"], s["new_rows"])
        kvb.load_kv4(s["pool"], s["read_rows"])
        return {"k": s["k_out"], "v": s["v_out"]}
    if op == "attend":
        kvb.launch_attention_kv4(s["pool"], s["query"], s["workspace"], s["out"], s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if op == "weigh":
        kvb.accumulate_weights_kv4(s["pool"], s["query"], s["lse"], s["weights"])
        return {"weights": s["weights"]}
    kvb.select_tokens(s["plan"], s["keep"], s["new_lens"])
    kvb.compact_kv4(s["pool"], s["plan"], s["keep"], s["new_table"], s["new_weights"])
    return _evicted(s, s["keep"], s["new_lens"], s["new_weights"])


def run(state):
    if own:
        return _own_pass(state)
    return {"store": _plain_store, "attend": _plain_attend, "weigh": _plain_weigh,
            "evict": _plain_evict}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return {"k": _exact_store(s["k_new"]), "v": _exact_store(s["v_new"])}
    if case["op"] == "evict":
        return None  # copies and choices: nothing is computed
    out, lse, weights = [], [], []
    for b in range(case["batch"]):
        o, z, w = _exact_sequence(s, b, int(s["lens"][b]))
        out.append(o)
        lse.append(z)
        weights.append(w)
    if case["op"] == "attend":
        return {"out": torch.stack(out), "lse": torch.stack(lse)}
    return {"weights": torch.stack(weights)}


def _exact_store(x):
    x = x.double()
    low = x.min(-1, keepdim=True).values
    scale = ((x.max(-1, keepdim=True).values - low) / 15).float().double()  # held in 32 bits
    code = torch.nan_to_num((x - low) / scale, nan=0.0).round().clamp(0, 15)
    return low + scale * code


def _exact_rows(s, what, b, h, n):
    """The first n K or V rows of sequence b and KV head h, in 64 bits."""
    pages = s["table"][b, :-(-n // s["case"]["page"])].long()
    code = s[what][pages, h]
    code = (code if what == "k" else code.mT).reshape(-1, s["case"]["dim"] // 2)[:n]
    pairs = s[what + "_params"][pages, h].reshape(-1, 2)[:n].double()
    even, odd = torch.remainder(code, 16).double(), torch.div(code, 16, rounding_mode="floor").double()
    rows = torch.empty((n, s["case"]["dim"]), dtype=torch.float64, device=code.device)
    rows[:, 0::2], rows[:, 1::2] = even, odd
    return rows * pairs[:, 0:1] + pairs[:, 1:2]


def _exact_sequence(s, b, n):
    case = s["case"]
    rows, group = case["rows"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros((rows, case["q_heads"], case["dim"]), dtype=torch.float64, device=DEVICE)
    lse = torch.full((rows, case["q_heads"]), -math.inf, dtype=torch.float64, device=DEVICE)
    weights = torch.zeros((case["kv_heads"], case["high"]), dtype=torch.float64, device=DEVICE)
    if case["op"] == "weigh":
        weights += s["weights"][b].double()
    for h in range(case["kv_heads"]):
        k = _exact_rows(s, "k", b, h, n)
        v = _exact_rows(s, "v", b, h, n) if case["op"] == "attend" else None
        if s["positions"] is None:
            at = torch.arange(n, device=DEVICE)
        else:
            pages = s["table"][b, :-(-n // case["page"])].long()
            at = s["positions"][pages, h].reshape(-1)[:n].long()
        for r in range(rows):
            here = n - rows + r if s["positions"] is None else int(s["q_positions"][b, r])
            visible = (at <= here) & (at > here - case["window"]) if case["window"] else at <= here
            if case["prefix"]:
                visible = visible | (at < case["prefix"])
            if not bool(visible.any()):
                continue
            heads = slice(h * group, (h + 1) * group)
            score = s["q"][b, r, heads].double() @ k.T * s["scale"]
            if case["softcap"]:
                score = torch.tanh(score / case["softcap"]) * case["softcap"]
            if s["slopes"] is not None:
                score = score - s["slopes"][heads].double()[:, None] * (here - at).abs()
            if case["op"] == "weigh":
                part = torch.exp(score - s["lse"][b, r, heads].double()[:, None])
                weights[h, :n] += torch.where(visible, part, 0.0).sum(0)
                continue
            score = score.masked_fill(~visible, -math.inf)
            lse[r, heads] = torch.logsumexp(score, -1)
            out[r, heads] = torch.softmax(score, -1) @ v
    return out, lse, weights
