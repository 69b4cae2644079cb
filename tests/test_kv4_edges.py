"""The 4-bit cache where its arithmetic and its checks can go wrong: queries
whose values share a sign, at bounds of the digits that the kernels hold."""
from __future__ import annotations

import ctypes
import json
import subprocess
import sys
from dataclasses import replace
from pathlib import Path

import numpy as np
import pytest
import torch

import kvbridge_b200 as kvb
from kvbridge_b200 import _lib

import kv4_testutil as util
from kv4_testutil import EPS, ROUND, SMALLEST, Rule, make_cache


def bounds(cache, rule, want):
    """What the kernels' formats allow around util.expected (causal by index):

    * scores: queries are fixed point with a unit of at most 2^-21 of the row's
      largest value, for every type: half of it, scale * max|q| * sum|k| * 2^-22;
      the fp32 fold of scale_t * (q . code) and lo * sum q a few 2^-24 of scale *
      sum|q| * max|k|, the score's own roundings 8 * 2^-24 of it.
    * sums of n probabilities in fp32, a quarter of the tokens a lane: n / 4 + 16
      roundings; exp 2^-21.
    * probability times V scale: half a unit, 2^-16 (fp32 outputs 2^-23) of the
      largest of its 64 tokens, times a code's distance from 8.
    * the result's own rounding.

    Returns the bounds of out, lse and weights."""
    scale, group = cache.dim ** -0.5, rule.group
    out, lse = np.zeros_like(want.out), np.zeros_like(want.lse)
    weights = [np.zeros_like(w) for w in want.weights]
    grain = 2.0 ** (-23 if rule.dtype == torch.float32 else -16)
    for b, n in enumerate(cache.lens):
        sums = (n / 4 + 16) * EPS + 2.0 ** -21
        for h in range(cache.heads):
            k, v = cache.dense("k", b, h), cache.dense("v", b, h)
            t = np.arange(n)
            par = cache.v_params.numpy()[cache.table[b].numpy()[t // cache.page], h, t % cache.page].astype(np.float64)
            for r in range(rule.rows):
                see = t <= n - rule.rows + r
                if not see.any():
                    continue
                for head in range(h * group, (h + 1) * group):
                    q = rule.q[b, r, head].double().numpy()
                    x = scale * (k[see] @ q)
                    score = scale * np.abs(q).max() * np.abs(k[see]).sum(-1).max() * 2.0 ** -22
                    score += 16 * EPS * scale * np.abs(q).sum() * np.abs(k[see]).max() + 8 * EPS * np.abs(x).max()
                    p = np.exp(x - want.lse[b, r, head])
                    lse[b, r, head] = score + sums + 4 * EPS * abs(want.lse[b, r, head])
                    weights[b][h, see] += p * (2 * score + sums + 2 * lse[b, r, head])
                    held = np.zeros(n)
                    held[see] = p * par[see, 0]
                    tiles = sum(8 * grain * held[i:i + 64].max() * see[i:i + 64].sum() for i in range(0, n, 64))
                    parts = (p[:, None] * (np.abs(v[see]) + 16 * par[see, :1])).sum(0)
                    own = want.out[b, r, head]
                    out[b, r, head] = ((2 * score + 2 * sums) * parts + tiles
                                       + ROUND[rule.dtype] * np.abs(own) + SMALLEST[rule.dtype])
    return out, lse, weights


def signed_queries(shape, dtype, seed):
    """One kind of query values a sequence, most with a mean far from zero."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(shape, generator=g)
    q[0], q[1], q[2], q[3], q[4] = 1.0, -1.0, 1.5, 1.99, -1.99
    q[5] = torch.rand(shape[1:], generator=g)
    q[6] += 1
    q[7] += 3
    q[8] = -0.25 - 0.5 * torch.rand(shape[1:], generator=g)
    return q.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("rows,group", [(1, 1), (1, 4), (1, 8), (3, 4)])
def test_queries_with_a_mean(cuda_device, dtype, dim, page, rows, group):
    """Output, log-sum-exp and weights: a query's sum multiplies every token's offset."""
    lens = [130, 64, 70, 200, 65, 129, 128, 90, 193, 150]
    cache = make_cache(lens, 2, dim, page, seed=5)
    rule = Rule(rows=rows, group=group, dtype=dtype)
    rule.q = signed_queries((len(lens), rows, 2 * group, dim), dtype, 6)
    want = util.expected(cache, rule)
    out_tol, lse_tol, weight_tol = bounds(cache, rule, want)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    out, lse = util.attend(cache, rule, cuda_device, pool=pool, query=query)
    for b in range(len(lens)):
        assert np.all(np.abs(lse[b] - want.lse[b]) <= lse_tol[b]), (b, np.abs(lse[b] - want.lse[b]).max(), lse_tol[b].max())
        assert np.all(np.abs(out[b] - want.out[b]) <= out_tol[b]), (b, np.abs(out[b] - want.out[b]).max(), out_tol[b].max())
    weights = torch.zeros((len(lens), 2, max(lens)), device=cuda_device)
    kvb.accumulate_weights_kv4(pool, query, torch.from_numpy(want.lse).float().to(cuda_device), weights)
    got = weights.cpu().double().numpy()
    for b, n in enumerate(lens):
        off = np.abs(got[b, :, :n] - want.weights[b])
        # (sums over the columns add a rounding each)
        assert np.all(off <= weight_tol[b] + rows * group * EPS * want.weights[b]), (b, off.max())


NO_PAGE = -1  # what an unassigned entry of an int32 block table usually holds


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("rule", [Rule(), Rule(group=8), Rule(window=150), Rule(slopes=True)], ids=str)
@pytest.mark.parametrize("bad", [NO_PAGE, 1 << 20, -7])
def test_every_bad_page_id_is_reported(cuda_device, page, rule, bad):
    """Any id that is not in the pool, -1 among them, inside a sequence; none beyond its end."""
    cache = make_cache([90, 250, 40], 1, 128, page, seed=41)
    rule = util.make_query(cache, rule, 42)
    for b, n in enumerate(cache.lens):
        cache.table[b, -(-n // page):] = bad
    # A window of 150 starts at token 100: the 64 tokens before its first stage are not looked at.
    for at, status in ((None, 0), (64, 4), (249, 4), (150, 4), (0, 0 if rule.window else 4)):
        table = cache.table.clone()
        if at is not None:
            cache.table[1, at // page] = bad
        pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
        cache.table = table
        kvb.read_device_status()
        util.attend(cache, rule, cuda_device, pool=pool, query=query)
        assert kvb.read_device_status() == status, at
        lse = torch.zeros(query.lse_shape, device=cuda_device)
        kvb.accumulate_weights_kv4(pool, query, lse, torch.zeros((3, 1, 250), device=cuda_device))
        assert kvb.read_device_status() == status, at


def without(cache, rule, dropped):
    """The cache and rule that stand for this call with the `dropped` (sequence,
    first token, end) hidden: positions that say what the indices did, beyond
    every row for the hidden tokens."""
    hidden = replace(cache)
    hidden.positions = torch.zeros(cache.k_params.shape[:-1], dtype=torch.int32)
    for b, n in enumerate(cache.lens):
        for h in range(cache.heads):
            at = torch.from_numpy(cache.token_positions(b, h)).int()
            for b2, first, end in dropped:
                if b2 == b:
                    at[first:end] = 1 << 30
            t = torch.arange(n)
            hidden.positions[cache.table[b].long()[t // cache.page], h, t % cache.page] = at
    rule = replace(rule)
    if rule.q_positions is None:
        rule.q_positions = torch.tensor([[n - rule.rows + r for r in range(rule.rows)] for n in cache.lens], dtype=torch.int32)
    return hidden, rule


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 32), (256, 64), (128, 64)])
@pytest.mark.parametrize("rule,positions", [
    (Rule(), False), (Rule(group=8, dtype=torch.float32), False), (Rule(rows=3, group=3, window=150), False),
    (Rule(window=90, prefix=[20, 70, 0, 300, 100]), False), (Rule(group=5, prefix=[0, 250, 400, 9, 1000]), False),
    (Rule(softcap=20.0, slopes=True, rows=2), False), (Rule(rows=2), True), (Rule(group=8, slopes=True, window=300), True),
], ids=str)
@pytest.mark.parametrize("bound", [None, 4000])
def test_tokens_of_a_bad_page_are_not_seen(cuda_device, dim, page, rule, positions, bound):
    """First, inner, last and all pages of a sequence: attention, log-sum-exp
    and weights are those without the page's tokens, whatever a warp read before."""
    lens = [100, 333, 600, 64, 1500]
    cache = make_cache(lens, 2, dim, page, seed=51, positions=positions)
    rule = util.make_query(cache, rule, 52)
    drop = [(0, 0), (1, 64 // page), (1, 333 // page), (2, 128 // page), (2, 128 // page + 1), (4, 3), (4, 1000 // page)]
    drop += [(3, j) for j in range(64 // page)]  # the whole sequence
    hidden, plain = without(cache, rule, [(b, j * page, (j + 1) * page) for b, j in drop])
    want = util.expected(hidden, plain)
    table = cache.table.clone()
    for i, (b, j) in enumerate(drop):
        table[b, j] = (NO_PAGE, 1 << 20, cache.k.shape[0])[i % 3]
    good, cache.table = cache.table, table
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device, max_tokens=bound)
    cache.table = good
    kvb.read_device_status()
    out, lse = util.attend(cache, rule, cuda_device, pool=pool, query=query)
    assert kvb.read_device_status() == 4
    empty = np.isneginf(want.lse)
    assert np.all(empty[3]) and np.array_equal(empty, np.isneginf(lse)) and np.all(out[empty] == 0)
    assert np.all(np.abs(lse[~empty] - want.lse[~empty]) <= want.lse_tol[~empty])
    assert np.all(np.abs(out - want.out) <= want.out_tol)
    start = torch.rand((len(lens), 2, 4000))
    weights = start.to(cuda_device)
    kvb.accumulate_weights_kv4(pool, query, torch.from_numpy(want.lse).float().to(cuda_device), weights)
    assert kvb.read_device_status() == 4
    got, start = weights.cpu().double().numpy(), start.double().numpy()
    for b, n in enumerate(lens):
        full = start[b, :, :n] + want.weights[b]
        assert np.all(np.abs(got[b, :, :n] - full) <= want.weight_tol[b] + 4 * EPS * full)
    for b, j in drop:
        assert np.array_equal(got[b, :, j * page:(j + 1) * page], start[b, :, j * page:(j + 1) * page])


@pytest.mark.gpu
def test_short_sequences_with_bad_pages(cuda_device):
    """Calls of one warp a segment: each of 40 sequences lacks another page."""
    lens = [1 + (i * 29) % 128 for i in range(40)]
    cache = make_cache(lens, 2, 128, 16, seed=53)
    rule = util.make_query(cache, Rule(rows=2, group=2), 54)
    drop = [(b, (b * 5) % -(-n // 16)) for b, n in enumerate(lens)]
    hidden, plain = without(cache, rule, [(b, 16 * j, 16 * j + 16) for b, j in drop])
    want = util.expected(hidden, plain)
    for b, j in drop:
        cache.table[b, j] = NO_PAGE
    out, lse = util.attend(cache, rule, cuda_device)
    assert kvb.read_device_status() == 4
    empty = np.isneginf(want.lse)
    assert np.array_equal(empty, np.isneginf(lse)) and np.all(out[empty] == 0)
    assert np.all(np.abs(lse[~empty] - want.lse[~empty]) <= want.lse_tol[~empty])
    assert np.all(np.abs(out - want.out) <= want.out_tol)


@pytest.mark.gpu
@pytest.mark.parametrize("rule", [Rule(rows=4), Rule(window=60, group=8), Rule(window=60, rows=3, softcap=30.0)], ids=str)
@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("batch", [3, 34])
def test_negative_prefixes_are_none(cuda_device, rule, positions, batch):
    """A negative int32 prefix shows nothing more and is reported; the others hold."""
    lens = [(180 + 77 * b) % 400 for b in range(batch)]
    cache = make_cache(lens, 1, 64, 16, seed=61, positions=positions)
    rule = util.make_query(cache, replace(rule, prefix=[(-1, 70, -(1 << 31))[b % 3] for b in range(batch)]), 62)
    valid = replace(rule, prefix=[max(x, 0) for x in rule.prefix])
    want = util.expected(cache, valid)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    kvb.read_device_status()
    out, lse = util.attend(cache, rule, cuda_device, pool=pool, query=query)
    assert kvb.read_device_status() == 5
    empty = np.isneginf(want.lse)
    assert np.array_equal(empty, np.isneginf(lse))
    assert np.all(np.abs(lse[~empty] - want.lse[~empty]) <= want.lse_tol[~empty])
    assert np.all(np.abs(out - want.out) <= want.out_tol)
    weights = torch.zeros((batch, 1, max(lens)), device=cuda_device)
    kvb.accumulate_weights_kv4(pool, query, torch.from_numpy(want.lse).float().to(cuda_device), weights)
    assert kvb.read_device_status() == 5
    got = weights.cpu().double().numpy()
    for b, n in enumerate(lens):
        assert np.all(np.abs(got[b, :, :n] - want.weights[b]) <= want.weight_tol[b] + 4 * EPS * want.weights[b])
    check = util.device_query(cache, valid, cuda_device)
    util.attend(cache, valid, cuda_device, pool=pool, query=check)
    assert kvb.read_device_status() == 0


def test_eviction_in_place_is_refused(kvb_lib):
    """Lengths and weights are read by CTAs that run beside the one that writes
    their successors, so these may not share memory. No call here gets to a launch."""
    base = 0x10000000  # never dereferenced
    pool = _lib.KvbKv4Pool(3, 64, 16, 100, *[base] * 4, None)
    plan = _lib.KvbKv4Eviction(2, 3, 200, 96, 4, 16, base, base, 256)

    def select(kept_lens):
        return kvb_lib.kvb_select_tokens(ctypes.byref(plan), base + 4096, kept_lens, None), _lib.last_error()

    def compact(new_weights, stride):
        return kvb_lib.kvb_compact_kv4(ctypes.byref(pool), ctypes.byref(plan), base, 16, base, base, 8, new_weights, stride,
                                       None), _lib.last_error()

    for at in (-4, 0, 4):
        assert select(base + at) == (_lib.KVB_EINVAL, "kept_lens must not overlap seq_lens")
    row = 4 * 256
    overlapping = [(base, 256), (base + 4 * 199, 256), (base - 4 * 95, 96), (base + 4 * 200, 257), (base + 4 * 161, 256),
                   (base + 5 * row + 4 * 199, 96), (base - 5 * row, 256), (base - 4 * 480 - 4 * 95, 96)]
    for at, stride in overlapping:
        assert compact(at, stride) == (_lib.KVB_EINVAL, "new_weights must not overlap weights"), (at - base, stride)


@pytest.mark.gpu
def test_compaction_into_the_same_rows_beside_the_weights(cuda_device):
    """Rows that hold the old weights and then the new ones share no float: allowed."""
    lens, heads, budget = [150, 200], 3, 96
    cache = make_cache(lens, heads, 64, 16, seed=71, spare=12)
    pool, device = cache.to(cuda_device), cuda_device
    both = torch.rand((2, heads, 400), device=device)
    before = both.clone()
    free = [p for p in range(pool.pages) if p not in cache.table[0, :10].tolist() + cache.table[1, :13].tolist()]
    new_table = torch.tensor(free[:12], dtype=torch.int32, device=device)
    table, seq_lens = cache.table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)
    keep = torch.empty((2, heads, budget), dtype=torch.int32, device=device)
    kept = torch.empty(2, dtype=torch.int32, device=device)
    plan = _lib.KvbKv4Eviction(2, heads, 200, budget, 4, 16, seq_lens.data_ptr(), both.data_ptr(), 400)
    lib = _lib.load()
    torch.cuda.synchronize()
    _lib.check(lib.kvb_select_tokens(ctypes.byref(plan), keep.data_ptr(), kept.data_ptr(), None))
    _lib.check(lib.kvb_compact_kv4(pool._ref, ctypes.byref(plan), table.data_ptr(), table.shape[1], keep.data_ptr(),
                                   new_table.data_ptr(), 6, both.data_ptr() + 4 * 200, 400, None))
    torch.cuda.synchronize()
    assert torch.equal(both[..., :200], before[..., :200]) and torch.equal(both[..., 296:], before[..., 296:])
    assert torch.equal(both[..., 200:296], before.gather(-1, keep.long()))


COUNT_COPIES = """
import json, warnings
import torch
from torch.profiler import ProfilerActivity, profile
import kvbridge_b200 as kvb

def copies():
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with profile(activities=[ProfilerActivity.CUDA]) as p:
            status = kvb.read_device_status()
            torch.cuda.synchronize()
    count = {e.key: e.count for e in p.key_averages()}
    return [status, count.get("cudaMemcpyFromSymbol", 0), count.get("cudaMemcpyToSymbol", 0)]

torch.zeros(1, device="cuda")
copies()
result = [copies()]
pool = kvb.Kv4Pool.empty(2, 1, 16, 64)
x = torch.zeros((1, 1, 64), device="cuda")
for slot in (3, 32):
    kvb.append_kv4(pool, kvb.Kv4Rows(x, x, torch.tensor([slot], device="cuda")))
    result.append(copies())
result.append(copies())
print(json.dumps(result))
"""


@pytest.mark.gpu
def test_reading_the_status_costs_no_more_than_its_words(cuda_device):
    """[status, copies from the device, copies to it]: one word where the 4-bit
    kernels have not run, two where they have, and a reset only of a code."""
    root = Path(__file__).resolve().parents[1]
    run = subprocess.run([sys.executable, "-c", COUNT_COPIES], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert json.loads(run.stdout.splitlines()[-1]) == [[0, 1, 0], [0, 2, 0], [6, 2, 1], [0, 2, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [1e-45, 1e-39, 1e-30, 1e30, 3e38])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_caps_at_the_ends_of_the_range(cuda_device, softcap, dtype):
    """Caps whose reciprocal overflows or vanishes, with queries that score 0 too."""
    cache = make_cache([70, 300], 2, 128, 64, seed=81)
    rule = util.make_query(cache, Rule(softcap=softcap, rows=2, dtype=dtype), 82)
    rule.q[0, 1] = 0
    rule.q[1, :, ::3] = 0
    out, lse = util.check_attention(cache, rule, cuda_device)
    assert np.all(np.isfinite(lse)) and np.all(np.isfinite(out))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (256, 64)])
@pytest.mark.parametrize("positions", [False, True])
def test_skipped_kept_tokens_leave_nan(cuda_device, dim, page, positions):
    """The new slot of a kept token that cannot be moved holds NaN and position 0,
    not what the page held before; the others are moved."""
    budget, heads = 150, 2
    cache = make_cache([400], heads, dim, page, seed=91, spare=2 * -(-budget // page), positions=positions)
    pool = cache.to(cuda_device)
    used = cache.table[0, :-(-400 // page)].tolist()
    new = [p for p in range(pool.pages) if p not in used][:-(-budget // page)]
    table = cache.table.clone()
    table[0, 2 * 64 // page] = NO_PAGE  # tokens from 128 on
    lens, kept = (torch.tensor([n], dtype=torch.int32, device=cuda_device) for n in (400, 0))
    weights = torch.rand((1, heads, 400), device=cuda_device)
    plan = kvb.EvictPlan(weights, lens, table.to(cuda_device), budget=budget, sinks=4, recent=20)
    keep = torch.empty((1, heads, budget), dtype=torch.int32, device=cuda_device)
    kvb.select_tokens(plan, keep, kept)
    keep[0, 0, 70], keep[0, 1, 3] = 400, -1  # beyond the sequence, and no token
    for name in ("k_params", "v_params"):
        getattr(pool, name)[torch.tensor(new, device=cuda_device)] = 0.5
    kvb.read_device_status()
    kvb.compact_kv4(pool, plan, keep, torch.tensor([new], dtype=torch.int32, device=cuda_device))
    assert kvb.read_device_status() == 8
    at = torch.arange(budget)
    pages, slots = torch.tensor(new)[at // page], at % page
    for h in range(heads):
        t = keep[0, h].cpu().long()
        gone = (t < 0) | (t >= 400) | (t // page == 2 * 64 // page)
        assert bool(gone.any()) and not bool(gone.all())
        source = table[0].long()[t.clamp(0, 399) // page], h, t.clamp(0, 399) % page
        for name in ("k_params", "v_params"):
            got = getattr(pool, name).cpu()[pages, h, slots]
            assert torch.isnan(got[gone]).all()
            assert torch.equal(got[~gone], getattr(cache, name)[source][~gone])
        if positions:
            want = torch.where(gone, 0, cache.positions[source])
            assert torch.equal(pool.positions.cpu()[pages, h, slots], want)
    last = budget % page  # nothing is written past the kept tokens
    assert torch.all(pool.k_params[new[-1], :, last:] == 0.5) and torch.all(pool.v_params[new[-1], :, last:] == 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("wrong", [None, [[0, 1]], torch.zeros((2, 3), dtype=torch.int32)], ids=["none", "list", "host"])
def test_what_is_no_cuda_tensor_raises_value_errors(cuda_device, wrong):
    cache = make_cache([70], 1, 64, 16, seed=95)
    rule = util.make_query(cache, Rule(group=1), 96)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    lens = torch.tensor([70], dtype=torch.int32, device=cuda_device)
    lse, table = torch.zeros(query.lse_shape, device=cuda_device), cache.table.to(cuda_device)
    plan = kvb.EvictPlan(torch.rand((1, 1, 70), device=cuda_device), lens, table, budget=16)
    keep = torch.zeros((1, 1, 16), dtype=torch.int32, device=cuda_device)
    for call in (
        lambda: kvb.Kv4Query(rule.q.to(cuda_device), lens, wrong, 70, 1, 0.1),
        lambda: kvb.Kv4Query(rule.q.to(cuda_device), wrong, table, 70, 1, 0.1),
        lambda: kvb.EvictPlan(plan.weights, lens, wrong, budget=16),
        lambda: kvb.accumulate_weights_kv4(pool, query, lse, wrong),
        lambda: kvb.accumulate_weights_kv4(pool, query, wrong, plan.weights),
        lambda: kvb.compact_kv4(pool, plan, keep, wrong),
        lambda: kvb.compact_kv4(pool, plan, keep, table, [0.0]),
        lambda: kvb.launch_attention_kv4(pool, query, wrong, torch.empty_like(query.q)),
    ):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def spread(x, offset, extra):
    """x [tokens, ..] as a view whose tokens lie `extra` elements further apart, from `offset` on."""
    row = x[0].numel()
    flat = torch.zeros(offset + len(x) * (row + extra), dtype=x.dtype, device=x.device)
    return flat.as_strided(x.shape, (row + extra,) + x[0].stride(), offset).copy_(x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("offset,extra", [(1, 0), (0, 1), (3, 5), (8, 4)])
def test_rows_queries_and_outputs_off_16_bytes(cuda_device, dtype, offset, extra):
    """Elements' own alignment is enough for rows, queries and outputs, and strides may be odd."""
    cache = make_cache([130, 70, 300], 2, 128, 32, seed=101)
    rule = util.make_query(cache, Rule(rows=2, group=4, dtype=dtype), 102)
    want = util.expected(cache, rule)
    pool, plain = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    q = spread(rule.q.to(cuda_device).flatten(0, 1), offset, extra)  # batch and row strides
    q = q.as_strided(rule.q.shape, (2 * q.stride(0),) + q.stride(), offset)
    query = kvb.Kv4Query(q, *plain._kept[:2], max_tokens=300, kv_heads=2, scale=128 ** -0.5)
    space = torch.empty(kvb.attention_kv4_workspace_bytes(pool, query), dtype=torch.uint8, device=cuda_device)
    out, same = torch.full((q.numel() + 16,), np.nan, dtype=dtype, device=cuda_device), torch.empty_like(plain.q)
    kvb.launch_attention_kv4(pool, query, space, out[offset:offset + q.numel()].view(q.shape))
    kvb.launch_attention_kv4(pool, plain, space, same)
    assert torch.equal(out[offset:offset + q.numel()].view(q.shape), same)
    assert torch.isnan(out[:offset]).all() and torch.isnan(out[offset + q.numel():]).all()
    assert np.all(np.abs(same.double().cpu().numpy() - want.out) <= want.out_tol)

    g = torch.Generator().manual_seed(103)
    k, v = (torch.randn((100, 2, 128), generator=g).to(dtype).to(cuda_device) for _ in range(2))
    slots = (torch.arange(100) + 7).to(cuda_device)
    pools = [kvb.Kv4Pool.empty(4, 2, 32, 128, device=cuda_device) for _ in range(2)]
    for p in pools:
        for x in (p.k, p.v, p.k_params, p.v_params):
            x.zero_()
    kvb.append_kv4(pools[0], kvb.Kv4Rows(k, v, slots))
    kvb.append_kv4(pools[1], kvb.Kv4Rows(spread(k, offset, extra), spread(v, 2 * offset, extra), slots))
    for name in ("k", "v", "k_params", "v_params"):
        assert torch.equal(getattr(pools[0], name), getattr(pools[1], name))
    dense = [torch.empty_like(k) for _ in range(2)]
    kvb.load_kv4(pools[0], kvb.Kv4Rows(*dense, slots))
    apart = [spread(torch.zeros_like(k), offset, extra), spread(torch.zeros_like(v), offset, extra)]
    kvb.load_kv4(pools[0], kvb.Kv4Rows(*apart, slots))
    assert torch.equal(dense[0], apart[0]) and torch.equal(dense[1], apart[1])
