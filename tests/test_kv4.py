"""The 4-bit paged cache: refusals (CPU), and the kernels against 64-bit
restatements of the formulas (GPU)."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

import kvbridge_b200 as kvb
from kvbridge_b200 import _lib

import kv4_testutil as util
from kv4_testutil import Rule, check_attention, make_cache, make_query

FAKE = 0x10000  # never dereferenced


# ---------------------------------------------------------------------------
# Refusals: nothing here reaches a GPU.


def c_pool(**kw):
    base = dict(kv_heads=8, dim=128, page_tokens=64, pages=16, k=FAKE, v=FAKE, k_params=FAKE, v_params=FAKE, positions=None)
    base.update(kw)
    return _lib.KvbKv4Pool(*(base[n] for n, _ in _lib.KvbKv4Pool._fields_))


def c_query(**kw):
    base = dict(batch=2, rows=1, q_heads=32, table_stride=8, max_tokens=512, type=1, scale=0.1, softcap=0.0, window=0, q=FAKE,
                batch_stride=4096, row_stride=4096, seq_lens=FAKE, block_table=FAKE, q_positions=None, slopes=None,
                prefix_lens=None)
    base.update(kw)
    return _lib.KvbKv4Query(*(base[n] for n, _ in _lib.KvbKv4Query._fields_))


def c_rows(**kw):
    base = dict(tokens=3, type=2, k=FAKE, v=FAKE, k_stride=1024, v_stride=1024, slots=FAKE, positions=None)
    base.update(kw)
    return _lib.KvbKv4Rows(*(base[n] for n, _ in _lib.KvbKv4Rows._fields_))


def c_eviction(**kw):
    base = dict(batch=2, kv_heads=8, max_tokens=512, budget=128, sinks=4, recent=16, seq_lens=FAKE, weights=FAKE,
                weight_stride=512)
    base.update(kw)
    return _lib.KvbKv4Eviction(*(base[n] for n, _ in _lib.KvbKv4Eviction._fields_))


def refuses(status, text):
    assert status == _lib.KVB_EINVAL
    assert text in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(kv_heads=0), "kv_heads"), (dict(dim=96), "dim 64, 128 or 256"), (dict(page_tokens=48), "page_tokens"),
    (dict(pages=0), "pages"), (dict(pages=1 << 31, kv_heads=64), "extent"),
])
def test_pool_refusals(kvb_lib, kw, text):
    refuses(kvb_lib.kvb_append_kv4(ctypes.byref(c_pool(**kw)), ctypes.byref(c_rows()), None), text)
    assert text in kvb_lib.kvb_kv4_pool_error(ctypes.byref(c_pool(**kw))).decode()
    refuses(kvb_lib.kvb_launch_attention_kv4(ctypes.byref(c_pool(**kw)), ctypes.byref(c_query()), FAKE, 1 << 30, FAKE, FAKE,
                                             None), text)


def test_rows_refusals(kvb_lib):
    for call in (kvb_lib.kvb_append_kv4, kvb_lib.kvb_load_kv4):
        def run(pool=None, **kw):
            return call(ctypes.byref(pool or c_pool()), ctypes.byref(c_rows(**kw)), None)

        refuses(run(type=3), "element type")
        refuses(run(k=None), "non-null")
        refuses(run(slots=FAKE + 4), "aligned")
        refuses(run(v=FAKE + 1), "aligned")
        refuses(run(k_stride=1023), "strides")
        refuses(run(v_stride=-5), "strides")
        refuses(run(c_pool(v_params=FAKE + 8)), "16-byte")
        refuses(run(c_pool(k=None)), "non-null")
        refuses(call(None, ctypes.byref(c_rows()), None), "pool pointer")
        refuses(call(ctypes.byref(c_pool()), None, None), "rows pointer")
        assert run(tokens=0, k=None, v=None, slots=None) == _lib.KVB_OK  # nothing to do
    refuses(kvb_lib.kvb_append_kv4(ctypes.byref(c_pool(positions=FAKE)), ctypes.byref(c_rows()), None), "positions")


@pytest.mark.parametrize("kw,text", [
    (dict(batch=0), "positive"), (dict(rows=0), "positive"), (dict(q_heads=12), "divisible"),
    (dict(rows=33), "at most 128"), (dict(type=-1), "element type"), (dict(table_stride=0), "table_stride"),
    (dict(scale=math.nan), "scale"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=math.inf), "softcap"), (dict(batch=65536), "65535"), (dict(row_stride=-1), "strides"),
    (dict(max_tokens=0x7fffffff), "2^31"),
])
def test_query_refusals(kvb_lib, kw, text):
    pool = c_pool()
    q = c_query(**kw)
    size = ctypes.c_size_t()
    assert text in kvb_lib.kvb_kv4_query_error(ctypes.byref(pool), ctypes.byref(q)).decode()
    refuses(kvb_lib.kvb_attention_kv4_workspace_bytes(ctypes.byref(pool), ctypes.byref(q), ctypes.byref(size)), text)
    refuses(kvb_lib.kvb_launch_attention_kv4(ctypes.byref(pool), ctypes.byref(q), FAKE, 1 << 40, FAKE, None, None), text)
    refuses(kvb_lib.kvb_accumulate_weights_kv4(ctypes.byref(pool), ctypes.byref(q), FAKE, FAKE, 1 << 40, None), text)


def test_attention_buffer_refusals(kvb_lib):
    def run(pool=None, ws=FAKE, size=1 << 40, out=FAKE, lse=FAKE, **kw):
        return kvb_lib.kvb_launch_attention_kv4(ctypes.byref(pool or c_pool()), ctypes.byref(c_query(**kw)), ws, size, out,
                                                lse, None)

    refuses(run(q=None), "non-null")
    refuses(run(block_table=None), "non-null")
    refuses(run(q=FAKE + 1), "aligned")
    refuses(run(seq_lens=FAKE + 2), "aligned")
    refuses(run(slopes=FAKE + 2), "aligned")
    refuses(run(c_pool(positions=FAKE)), "q_positions")
    refuses(run(ws=None), "non-null")
    refuses(run(out=None), "non-null")
    refuses(run(ws=FAKE + 8), "16-byte")
    refuses(run(out=FAKE + 1), "elements")
    refuses(run(lse=FAKE + 2), "elements")

    def weigh(lse=FAKE, weights=FAKE, stride=512, **kw):
        return kvb_lib.kvb_accumulate_weights_kv4(ctypes.byref(c_pool()), ctypes.byref(c_query(**kw)), lse, weights, stride,
                                                  None)

    refuses(weigh(lse=None), "non-null")
    refuses(weigh(weights=FAKE + 2), "aligned")
    refuses(weigh(stride=511), "weight_stride")
    assert weigh(max_tokens=0) == _lib.KVB_OK  # no token can be weighed


@pytest.mark.parametrize("kw,text", [
    (dict(batch=0), "batch"), (dict(kv_heads=0), "kv_heads"), (dict(budget=0), "budget"),
    (dict(sinks=100, recent=29), "sinks + recent"), (dict(weight_stride=511), "weight_stride"),
    (dict(max_tokens=1 << 31, weight_stride=1 << 31), "2^31"), (dict(seq_lens=None), "non-null"),
    (dict(weights=FAKE + 1), "aligned"),
])
def test_eviction_refusals(kvb_lib, kw, text):
    e = c_eviction(**kw)
    refuses(kvb_lib.kvb_select_tokens(ctypes.byref(e), FAKE, FAKE, None), text)
    refuses(kvb_lib.kvb_compact_kv4(ctypes.byref(c_pool()), ctypes.byref(e), FAKE, 8, FAKE, FAKE, 8, None, 0, None), text)


def test_compaction_refusals(kvb_lib):
    def run(table=FAKE, width=8, keep=FAKE, new=FAKE, new_width=2, weights=None, stride=0, **kw):
        return kvb_lib.kvb_compact_kv4(ctypes.byref(c_pool()), ctypes.byref(c_eviction(**kw)), table, width, keep, new,
                                       new_width, weights, stride, None)

    refuses(run(kv_heads=4), "kv_heads differ")
    refuses(run(table=None), "non-null")
    refuses(run(keep=FAKE + 2), "aligned")
    refuses(run(width=0), "strides must be positive")
    refuses(run(new_width=1), "budget exceeds")
    refuses(run(weights=FAKE, stride=127), "new_weight_stride")
    refuses(kvb_lib.kvb_select_tokens(ctypes.byref(c_eviction()), None, FAKE, None), "non-null")


def test_python_layer_refuses_host_tensors(kvb_lib):
    x = torch.zeros((2, 3, 64))
    with pytest.raises(ValueError, match="CUDA tensor"):
        kvb.Kv4Rows(x, x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA tensor"):
        kvb.Kv4Pool.empty(2, 1, 16, 64, device="cpu")
    assert "launch_attention_kv4" in dir(kvb)
    with pytest.raises(AttributeError):
        kvb.no_such_name


# ---------------------------------------------------------------------------
# Append and read back


def store_rows(tokens, heads, dim, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, heads, dim), generator=g)
    x[::5] += 3
    x[1::7] *= 10
    if tokens > 8:
        x[3] = 0.75  # equal values: scale 0
        x[4] = 0.0
        x[5, :, :4] = torch.tensor([0.0, 15.0, 2.5, 3.5])  # ties to even
        x[5, :, 4:] = 0.0
        x[6, 0, 7] = math.inf
        x[7, 0, 1] = math.nan
        x[8, 0] = 1e-41 if dtype == torch.float32 else 0.0  # denormal
    return x.to(dtype)


def expected_pool(rows, slots, pool, page):
    """Writes quantised rows [tokens, heads, dim] into numpy pool arrays."""
    (kn, vn), (k, v, kp, vp) = rows, pool
    for x, code_pool, par_pool, is_v in ((kn, k, kp, False), (vn, v, vp, True)):
        code, par = util.quantize(x)
        code = util.pack(code)
        for t, slot in enumerate(slots):
            if 0 <= slot < k.shape[0] * page:
                at, s = slot // page, slot % page
                if is_v:
                    code_pool[at, :, :, s] = code[t]
                else:
                    code_pool[at, :, s] = code[t]
                par_pool[at, :, s] = par[t]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,heads,dim,page,layout", [
    (1, 1, 64, 16, "run"), (9, 3, 128, 32, "scattered"), (77, 2, 256, 64, "run"), (300, 8, 128, 64, "run"),
    (1000, 4, 64, 16, "run"), (333, 2, 128, 16, "scattered"), (200, 1, 256, 32, "pieces"), (130, 5, 64, 64, "pieces"),
])
def test_append_and_load(cuda_device, dtype, tokens, heads, dim, page, layout):
    kn, vn = store_rows(tokens, heads, dim, 1, dtype), store_rows(tokens, heads, dim, 2, dtype)
    g = torch.Generator().manual_seed(3)
    pages = -(-tokens // page) + 3
    order = torch.randperm(pages, generator=g)
    at = torch.arange(tokens) + 5
    slots = order[at // page] * page + at % page
    if layout == "scattered":
        slots = torch.randperm(pages * page, generator=g)[:tokens]
    if layout == "pieces":  # runs of different lengths with holes between them
        at = torch.arange(tokens) + torch.arange(tokens) // 7
        slots = at[at < pages * page]
        slots = torch.cat([slots, torch.full((tokens - len(slots),), -1)])
    if tokens > 2:
        slots[2] = -1
    host = [torch.randint(0, 256, (pages, heads, page, dim // 2), generator=g, dtype=torch.uint8),
            torch.randint(0, 256, (pages, heads, dim // 2, page), generator=g, dtype=torch.uint8),
            torch.randn((pages, heads, page, 2), generator=g), torch.randn((pages, heads, page, 2), generator=g)]
    pos = torch.full((pages, heads, page), -7, dtype=torch.int32)
    pool = kvb.Kv4Pool(*(x.to(cuda_device) for x in host), positions=pos.to(cuda_device))
    # rows are columns of a wider array
    wide = torch.randn((tokens, 2 * heads * dim + 8), device=cuda_device).to(dtype)
    kd = wide[:, 8:8 + heads * dim].unflatten(1, (heads, dim))
    vd = wide[:, 8 + heads * dim:].unflatten(1, (heads, dim))
    kd.copy_(kn)
    vd.copy_(vn)
    positions = torch.arange(tokens, dtype=torch.int32) * 3
    kvb.read_device_status()
    kvb.append_kv4(pool, kvb.Kv4Rows(kd, vd, slots.to(cuda_device), positions.to(cuda_device)))
    ko = torch.full((tokens, heads, dim), 7.0, dtype=dtype, device=cuda_device)
    vo = torch.full((tokens, heads, dim), 7.0, dtype=dtype, device=cuda_device)
    kvb.load_kv4(pool, kvb.Kv4Rows(ko, vo, slots.to(cuda_device)))
    torch.cuda.synchronize()
    assert kvb.read_device_status() == 0
    expected_pool((kn, vn), slots.tolist(), host, page)
    for t, slot in enumerate(slots.tolist()):
        if slot >= 0:
            pos[slot // page, :, slot % page] = positions[t]
    for name, want in zip(("k", "v", "k_params", "v_params"), host):
        assert np.array_equal(getattr(pool, name).cpu().numpy(), want.numpy(), equal_nan=want.is_floating_point()), name
    assert torch.equal(pool.positions.cpu(), pos)
    for got, x in ((ko, kn), (vo, vn)):
        code, par = util.quantize(x)
        value = par[..., 1:].double() + par[..., :1].double() * code.double()
        value[slots < 0] = 0
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(value))
        # one rounding of the exact value (an fma), then the rows' own
        tol = value.abs() * (util.ROUND[dtype] + util.EPS) + util.SMALLEST[dtype]
        ok = torch.isnan(value) | ((got - value).abs() <= tol)
        assert bool(ok.all())


@pytest.mark.gpu
def test_append_and_load_report_bad_slots(cuda_device):
    heads, dim, page, pages = 2, 128, 16, 2
    kn, vn = store_rows(4, heads, dim, 5, torch.float32), store_rows(4, heads, dim, 6, torch.float32)
    slots = torch.tensor([3, pages * page, 1 << 40, 17])
    host = [torch.zeros((pages, heads, page, dim // 2), dtype=torch.uint8),
            torch.zeros((pages, heads, dim // 2, page), dtype=torch.uint8),
            torch.zeros((pages, heads, page, 2)), torch.zeros((pages, heads, page, 2))]
    pool = kvb.Kv4Pool(*(x.to(cuda_device) for x in host))
    kvb.read_device_status()
    kvb.append_kv4(pool, kvb.Kv4Rows(kn.to(cuda_device), vn.to(cuda_device), slots.to(cuda_device)))
    assert kvb.read_device_status() == 6
    out = torch.full((4, heads, dim), 9.0, device=cuda_device)
    kvb.load_kv4(pool, kvb.Kv4Rows(out, torch.empty_like(out), slots.to(cuda_device)))
    assert kvb.read_device_status() == 6
    assert torch.all(out[1:3] == 0) and not torch.all(out[0] == 0)
    expected_pool((kn, vn), slots.tolist(), host, page)
    assert torch.equal(pool.k.cpu(), host[0]) and torch.equal(pool.v.cpu(), host[1])


# ---------------------------------------------------------------------------
# Attention


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 64), (128, 16), (128, 32), (128, 64), (256, 32), (256, 64)])
@pytest.mark.parametrize("group", [1, 4, 8])
def test_attention_ragged(cuda_device, dtype, dim, page, group):
    lens = [1, 63, 64, 65, 0, 200, 700]
    cache = make_cache(lens, 2, dim, page, seed=dim + page)
    check_attention(cache, make_query(cache, Rule(group=group, dtype=dtype), 7), cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,group,dtype", [
    (2, 1, torch.float16), (4, 2, torch.bfloat16), (3, 5, torch.float16), (8, 6, torch.float16), (7, 3, torch.float32),
    (1, 7, torch.float32), (1, 16, torch.bfloat16), (2, 64, torch.float16), (5, 1, torch.float32),
])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_rows_and_groups(cuda_device, rows, group, dtype, dim):
    # sequences shorter than `rows` leave their first rows without a token
    cache = make_cache([rows + 3, 2, 0, 129, 300], 2, dim, 32, seed=rows * 10 + group)
    out, lse = check_attention(cache, make_query(cache, Rule(rows=rows, group=group, dtype=dtype), 8), cuda_device)
    if rows > 2:
        assert np.all(np.isneginf(lse[1, :rows - 2])) and np.all(out[2] == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("rule", [
    Rule(softcap=20.0), Rule(slopes=True), Rule(window=70), Rule(window=1), Rule(window=100, prefix=[5, 0, 700, 3]),
    Rule(prefix=[9, 400, 0, 1], rows=4), Rule(softcap=5.0, slopes=True, window=130, prefix=[16] * 4, rows=3, group=3),
    Rule(softcap=30.0, slopes=True, rows=2, group=8, dtype=torch.bfloat16),
    Rule(softcap=30.0, slopes=True, window=4000, group=5, dtype=torch.float32),
], ids=str)
@pytest.mark.parametrize("dim,page", [(64, 32), (128, 64), (256, 16)])
def test_attention_rules(cuda_device, rule, dim, page):
    cache = make_cache([40, 333, 600, 2], 2, dim, page, seed=11)
    check_attention(cache, make_query(cache, rule, 12), cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("rule", [
    Rule(), Rule(rows=3, group=2, window=90), Rule(slopes=True, prefix=[3, 50, 0]), Rule(group=8, dtype=torch.float32),
], ids=str)
@pytest.mark.parametrize("page", [16, 64])
def test_attention_explicit_positions(cuda_device, rule, page):
    cache = make_cache([1, 200, 450], 3, 128, page, seed=13, positions=True)
    check_attention(cache, make_query(cache, rule, 14), cuda_device)


@pytest.mark.gpu
def test_attention_positions_before_the_tokens(cuda_device):
    """Rows that stand before every token see nothing, explicit positions in any order."""
    cache = make_cache([100], 1, 64, 16, seed=15, positions=True)
    rule = make_query(cache, Rule(rows=3, window=20), 16)
    rule.q_positions = torch.tensor([[-5, 100000, 60]], dtype=torch.int32)
    out, lse = check_attention(cache, rule, cuda_device)
    assert np.all(np.isneginf(lse[0, :2])) and np.all(np.isfinite(lse[0, 2]))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,lens", [(1, [5000]), (8, [4096]), (2, [30000, 1, 9000]), (1, [20000])])
def test_attention_long(cuda_device, heads, lens):
    """Sequences split over many CTAs, partials merged."""
    cache = make_cache(lens, heads, 128, 64, seed=17)
    check_attention(cache, make_query(cache, Rule(dtype=torch.float32), 18), cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [33, 300])
def test_attention_many_sequences(cuda_device, batch):
    lens = [(i * 37) % 150 for i in range(batch)]
    cache = make_cache(lens, 2, 64, 16, seed=19)
    check_attention(cache, make_query(cache, Rule(group=2), 20), cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("max_tokens", [700, 1000, 100000])
def test_attention_length_bound_and_strides(cuda_device, max_tokens):
    cache = make_cache([700, 3, 64], 2, 128, 16, seed=21)
    cache.table = torch.nn.functional.pad(cache.table, (0, 6250 - cache.table.shape[1]))
    rule = make_query(cache, Rule(rows=2, group=3), 22)
    a = check_attention(cache, rule, cuda_device, max_tokens=max_tokens, strided=True)
    b = check_attention(cache, rule, cuda_device, max_tokens=max_tokens)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])  # strides change nothing


@pytest.mark.gpu
def test_attention_nan_rows_stay_with_those_who_see_them(cuda_device):
    """A NaN K row reaches exactly the query rows that see it; a NaN V row the same."""
    for what in ("k_params", "v_params"):
        cache = make_cache([200], 1, 128, 64, seed=23)
        rule = make_query(cache, Rule(rows=4, group=2), 24)
        getattr(cache, what)[cache.table[0, 198 // 64].item(), 0, 198 % 64] = math.nan  # seen by rows 2 and 3
        out, lse = util.attend(cache, rule, cuda_device)
        want = util.expected(cache, rule)
        assert np.all(np.abs(out - want.out)[0, :2] <= want.out_tol[0, :2])
        assert np.all(np.isnan(out[0, 2:]))
        assert np.all(np.isnan(lse[0, 2:])) == (what == "k_params")


@pytest.mark.gpu
def test_attention_extreme_scores(cuda_device):
    """Large scores of one token, of the first tile or the last; rows of equal values; a query of zeros."""
    for at in (0, 70, 255):
        cache = make_cache([256], 1, 64, 16, seed=25)
        rule = make_query(cache, Rule(group=2, dtype=torch.float32), 26)
        rule.q[0, 0, 1] = 0
        page, s = cache.table[0, at // 16].item(), at % 16
        cache.k_params[page, 0, s] *= 40
        cache.k_params[page, 0, (s + 1) % 16] = torch.tensor([0.0, 1.5])
        check_attention(cache, rule, cuda_device)


@pytest.mark.gpu
def test_attention_streams_graph_and_repeat(cuda_device):
    """Another stream, a captured graph and a repeated call give the same bits."""
    cache = make_cache([5000, 70], 4, 128, 64, seed=27)
    rule = make_query(cache, Rule(), 28)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    ws = torch.empty(kvb.attention_kv4_workspace_bytes(pool, query), dtype=torch.uint8, device=cuda_device)
    outs = [torch.empty(query.shape, dtype=rule.dtype, device=cuda_device) for _ in range(4)]
    kvb.launch_attention_kv4(pool, query, ws, outs[0])
    kvb.launch_attention_kv4(pool, query, ws, outs[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kvb.launch_attention_kv4(pool, query, ws, outs[2], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kvb.launch_attention_kv4(pool, query, ws, outs[3])
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.gpu
def test_attention_reports_bad_pages_and_lengths(cuda_device):
    cache = make_cache([200, 90], 1, 64, 16, seed=29)
    rule = make_query(cache, Rule(group=2), 30)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device, max_tokens=150)
    kvb.read_device_status()
    got = util.attend(cache, rule, cuda_device, pool=pool, query=query)
    assert kvb.read_device_status() == 5
    cache.lens[0] = 150  # what a clamped length stands for
    want = util.expected(cache, rule)
    assert np.all(np.abs(got[0] - want.out) <= want.out_tol)
    cache.table[0, 3] = 1 << 20
    query = util.device_query(cache, rule, cuda_device)
    got = util.attend(cache, rule, cuda_device, pool=pool, query=query)
    assert kvb.read_device_status() == 4
    assert np.all(np.abs(got[0] - want.out)[1] <= want.out_tol[1])  # the other sequence is untouched


@pytest.mark.gpu
def test_attention_launch_failure_is_reported(cuda_device):
    cache = make_cache([50], 1, 64, 16, seed=31)
    rule = make_query(cache, Rule(group=2), 32)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    kvb.debug_fail_launch(1, 2)
    with pytest.raises(RuntimeError, match="out of memory"):
        util.attend(cache, rule, cuda_device, pool=pool, query=query)
    util.check_attention(cache, rule, cuda_device)


@pytest.mark.gpu
def test_attention_pool_beyond_32_bits(cuda_device):
    """K offsets past 2^32 bytes."""
    heads, dim, page = 8, 256, 64
    pages = (1 << 32) // (heads * page * dim // 2) + 40
    try:
        pool = kvb.Kv4Pool.empty(pages, heads, page, dim, device=cuda_device)
    except torch.cuda.OutOfMemoryError:
        pytest.skip("not enough device memory")
    cache = make_cache([500], heads, dim, page, seed=33, garbage=False)
    n = cache.k.shape[0]
    for name in ("k", "v", "k_params", "v_params"):
        getattr(pool, name)[pages - n:] = getattr(cache, name).to(cuda_device)
    rule = make_query(cache, Rule(group=2), 34)
    want = util.expected(cache, rule)
    cache.table += pages - n
    query = util.device_query(cache, rule, cuda_device)
    out, lse = util.attend(cache, rule, cuda_device, pool=pool, query=query)
    assert np.all(np.abs(out - want.out) <= want.out_tol)
    # and the rows read back through slots that pass 32 bits once scaled
    slots = cache.table[0, 0].long() * page + torch.arange(page)
    k, v = (torch.empty((page, heads, dim), device=cuda_device) for _ in range(2))
    kvb.load_kv4(pool, kvb.Kv4Rows(k, v, slots.to(cuda_device)))
    cache.table -= pages - n
    assert np.allclose(k[:, 3].cpu().numpy(), cache.dense("k", 0, 3)[:page], rtol=1e-6, atol=1e-6)
    assert np.allclose(v[:, 7].cpu().numpy(), cache.dense("v", 0, 7)[:page], rtol=1e-6, atol=1e-6)


# ---------------------------------------------------------------------------
# Accumulated weights


@pytest.mark.gpu
@pytest.mark.parametrize("rule", [
    Rule(group=1), Rule(), Rule(group=8, dtype=torch.bfloat16), Rule(rows=3, group=7, dtype=torch.float32),
    Rule(softcap=20.0, slopes=True, window=90, prefix=[4, 0, 100, 1, 1], rows=2), Rule(rows=2, group=64),
], ids=str)
@pytest.mark.parametrize("dim,page,positions", [(64, 16, False), (128, 64, False), (128, 32, True), (256, 64, False)])
def test_weights(cuda_device, rule, dim, page, positions):
    cache = make_cache([1, 130, 600, 0, 64], 2, dim, page, seed=41, positions=positions)
    rule = make_query(cache, rule, 42)
    want = util.expected(cache, rule)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    width = 613  # rows that are not aligned to anything
    start = torch.rand((5, 2, width))
    weights = start.to(cuda_device)
    lse = torch.from_numpy(want.lse).float().to(cuda_device)
    kvb.accumulate_weights_kv4(pool, query, lse, weights)
    got = weights.cpu().double().numpy()
    again = start.to(cuda_device)
    kvb.accumulate_weights_kv4(pool, query, lse, again)
    assert torch.equal(weights, again)
    for b, n in enumerate(cache.lens):
        assert np.array_equal(got[b, :, n:], start[b, :, n:].double().numpy())
        full = start[b, :, :n].double().numpy() + want.weights[b]
        assert np.all(np.abs(got[b, :, :n] - full) <= want.weight_tol[b] + 4 * util.EPS * full)


@pytest.mark.gpu
def test_weights_of_shared_pages_and_their_sum(cuda_device):
    """Two sequences on the same pages keep weights of their own; a step adds one per query row and head."""
    cache = make_cache([300], 2, 64, 32, seed=43)
    cache.table = cache.table.repeat(2, 1)
    cache.lens = [300, 170]
    rule = make_query(cache, Rule(group=4, dtype=torch.float32), 44)
    pool, query = cache.to(cuda_device), util.device_query(cache, rule, cuda_device)
    out, lse = util.attend(cache, rule, cuda_device, pool=pool, query=query)
    weights = torch.zeros((2, 2, 300), device=cuda_device)
    kvb.accumulate_weights_kv4(pool, query, torch.from_numpy(lse).float().to(cuda_device), weights)
    assert np.allclose(weights.sum(-1).cpu().numpy(), 4.0, rtol=1e-4)
    assert torch.all(weights[1, :, 170:] == 0)


# ---------------------------------------------------------------------------
# Eviction


def choose(weights, n, budget, sinks, recent):
    """Kept tokens of one sequence and head."""
    if n <= budget:
        return list(range(n))
    always = set(range(sinks)) | set(range(n - recent, n))
    key = lambda t: (0 if math.isnan(weights[t]) else 1, -weights[t] if not math.isnan(weights[t]) else 0, t)  # noqa: E731
    rest = sorted((t for t in range(n) if t not in always), key=key)
    return sorted(always | set(rest[:budget - sinks - recent]))


def run_select(weights, lens, budget, sinks, recent, device, table=None):
    B, H, _ = weights.shape
    table = torch.zeros((B, 1), dtype=torch.int32, device=device) if table is None else table
    plan = kvb.EvictPlan(weights.to(device), torch.tensor(lens, dtype=torch.int32, device=device), table, budget=budget,
                         sinks=sinks, recent=recent)
    keep = torch.full((B, H, budget), -1, dtype=torch.int32, device=device)
    kept = torch.full((B,), -1, dtype=torch.int32, device=device)
    kvb.select_tokens(plan, keep, kept)
    torch.cuda.synchronize()
    return plan, keep, kept


@pytest.mark.gpu
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (50, 4, 10), (50, 25, 25), (300, 0, 100),
                                                 (1000, 4, 64), (5000, 1, 1)])
@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
def test_select(cuda_device, budget, sinks, recent, kind):
    lens = [0, 1, 49, 50, 51, 301, 2047, 4099]
    g = torch.Generator().manual_seed(51)
    w = torch.exp(2 * torch.randn((len(lens), 2, 4101), generator=g))
    if kind == "ties":
        w = (w * 2).round().clamp(max=3)
    if kind == "special":
        for value in (math.inf, -math.inf, math.nan, 0.0, -0.0, -1.0, 1e-42):
            w[torch.rand(w.shape, generator=g) < 0.05] = value
    _, keep, kept = run_select(w, lens, budget, sinks, recent, cuda_device)
    assert kept.tolist() == [min(n, budget) for n in lens]
    keep = keep.cpu()
    for b, n in enumerate(lens):
        for h in range(2):
            want = choose(w[b, h].tolist(), n, budget, sinks, recent)
            assert keep[b, h].tolist() == want + [0] * (budget - len(want)), (b, h)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40000, 131071, 500001])
def test_select_long(cuda_device, n):
    g = torch.Generator().manual_seed(52)
    w = torch.rand((1, 2, n), generator=g)
    w[0, 1] = (w[0, 1] * 7).floor()  # long ties
    budget, sinks, recent = n // 5, 4, 1000
    _, keep, kept = run_select(w, [n], budget, sinks, recent, cuda_device)
    assert kept.tolist() == [budget]
    for h in range(2):
        assert keep[0, h].cpu().tolist() == choose(w[0, h].tolist(), n, budget, sinks, recent)


@pytest.mark.gpu
def test_select_clamps_lengths(cuda_device):
    w = torch.rand((1, 1, 100))
    kvb.read_device_status()
    _, keep, kept = run_select(w, [500], 10, 0, 0, cuda_device)
    assert kvb.read_device_status() == 5
    assert keep[0, 0].cpu().tolist() == choose(w[0, 0].tolist(), 100, 10, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("positions", [True, False])
def test_compact(cuda_device, dim, page, positions):
    lens, heads, budget = [1, 100, 700, 0, 333], 3, 150
    cache = make_cache(lens, heads, dim, page, seed=61, spare=0, positions=positions)
    each = -(-budget // page)
    n = cache.k.shape[0]
    grow = lambda x: torch.cat([x, torch.full((len(lens) * each + 1,) + x.shape[1:], 3, dtype=x.dtype)])  # noqa: E731
    for name in ("k", "v", "k_params", "v_params") + (("positions",) if positions else ()):
        setattr(cache, name, grow(getattr(cache, name)))
    pool = cache.to(cuda_device)
    before = {m: getattr(pool, m).clone() for m in ("k", "v", "k_params", "v_params")}
    new_table = (n + torch.randperm(len(lens) * each)).to(torch.int32).view(len(lens), each)
    w = torch.rand((len(lens), heads, 711))
    table = cache.table.to(cuda_device)
    plan, keep, kept = run_select(w, lens, budget, 2, 20, cuda_device, table)
    new_w = torch.full((len(lens), heads, budget + 5), -1.0, device=cuda_device)
    kvb.read_device_status()
    kvb.compact_kv4(pool, plan, keep, new_table.to(cuda_device), new_w)
    torch.cuda.synchronize()
    assert kvb.read_device_status() == 0
    for m, old in before.items():
        assert torch.equal(getattr(pool, m)[:n].view(torch.uint8), old[:n].view(torch.uint8))  # old pages are only read
        assert torch.equal(getattr(pool, m)[-1], old[-1])  # and nothing beside the new ones is written
    moved = util.Cache(pool.k.cpu(), pool.v.cpu(), pool.k_params.cpu(), pool.v_params.cpu(), new_table,
                       [min(x, budget) for x in lens], page, pool.positions.cpu() if positions else None)
    assert torch.all(new_w[..., budget:] == -1)
    for b in range(len(lens)):
        for h in range(heads):
            at = keep[b, h, :moved.lens[b]].cpu().numpy()
            for what in ("k", "v"):
                assert np.array_equal(moved.dense(what, b, h), cache.dense(what, b, h)[at])
            if positions:
                assert np.array_equal(moved.token_positions(b, h), cache.token_positions(b, h)[at])
            row = np.zeros(budget, dtype=np.float32)
            row[:len(at)] = w[b, h].numpy()[at]
            assert np.array_equal(new_w[b, h, :budget].cpu().numpy(), row)


@pytest.mark.gpu
def test_compact_reports_bad_kept_tokens_and_pages(cuda_device):
    cache = make_cache([100], 1, 64, 16, seed=62, spare=8)
    pool = cache.to(cuda_device)
    plan, keep, kept = run_select(torch.rand((1, 1, 100)), [100], 20, 0, 0, cuda_device, cache.table.to(cuda_device))
    free = [p for p in range(pool.pages) if p not in cache.table[0].tolist()]
    new = torch.tensor([free[:2]], dtype=torch.int32, device=cuda_device)
    bad = keep.clone()
    bad[0, 0, 5] = 4000
    kvb.read_device_status()
    kvb.compact_kv4(pool, plan, bad, new)
    assert kvb.read_device_status() == 8
    kvb.compact_kv4(pool, plan, keep, torch.full_like(new, pool.pages))
    assert kvb.read_device_status() == 4
    short = kvb.EvictPlan(plan.weights, torch.tensor([100], dtype=torch.int32, device=cuda_device),
                          plan.block_table[:, :3].contiguous(), budget=20)
    bad[0, 0, 5] = 3 * 16  # beyond the block table's row
    kvb.compact_kv4(pool, short, bad, new)
    assert kvb.read_device_status() == 8
    kvb.compact_kv4(pool, plan, keep, new)
    assert kvb.read_device_status() == 0


@pytest.mark.gpu
def test_decode_with_eviction(cuda_device):
    """Append, attend, weigh and evict as a serving loop does; attention over
    the compacted cache equals attention over the kept tokens."""
    heads, dim, page, group, n, budget = 2, 128, 32, 4, 260, 96
    g = torch.Generator().manual_seed(71)
    pool = kvb.Kv4Pool.empty(24, heads, page, dim, device=cuda_device, positions=True)
    table = torch.arange(9, dtype=torch.int32, device=cuda_device)[None]
    x = [torch.randn((n, heads, dim), generator=g).bfloat16().to(cuda_device) for _ in range(2)]
    at = torch.arange(n, device=cuda_device)
    kvb.append_kv4(pool, kvb.Kv4Rows(*x, table[0].long()[at // page] * page + at % page, at.to(torch.int32)))
    lens = torch.tensor([n], dtype=torch.int32, device=cuda_device)
    q = torch.randn((1, 1, heads * group, dim), generator=g).bfloat16().to(cuda_device)
    qpos = torch.tensor([[n]], dtype=torch.int32, device=cuda_device)
    common = dict(kv_heads=heads, scale=dim ** -0.5, window=0, q_positions=qpos)
    query = kvb.Kv4Query(q, lens, table, max_tokens=9 * page, **common)
    ws = torch.empty(kvb.attention_kv4_workspace_bytes(pool, query), dtype=torch.uint8, device=cuda_device)
    out, lse = torch.empty_like(q), torch.empty((1, 1, heads * group), device=cuda_device)
    weights = torch.zeros((1, heads, 9 * page), device=cuda_device)
    kvb.launch_attention_kv4(pool, query, ws, out, lse)
    kvb.accumulate_weights_kv4(pool, query, lse, weights)
    plan = kvb.EvictPlan(weights, lens, table, budget=budget, sinks=4, recent=16)
    keep = torch.empty((1, heads, budget), dtype=torch.int32, device=cuda_device)
    new_lens = torch.empty((1,), dtype=torch.int32, device=cuda_device)
    new_table = torch.arange(12, 12 + budget // page, dtype=torch.int32, device=cuda_device)[None]
    kvb.select_tokens(plan, keep, new_lens)
    kvb.compact_kv4(pool, plan, keep, new_table)
    after = kvb.Kv4Query(q, new_lens, new_table, max_tokens=budget, **common)
    kvb.launch_attention_kv4(pool, after, ws, out, lse)
    torch.cuda.synchronize()
    old = util.Cache(pool.k.cpu(), pool.v.cpu(), pool.k_params.cpu(), pool.v_params.cpu(), table.cpu(), [n], page)
    for h in range(heads):
        kept = keep[0, h].cpu().numpy()
        k, v = old.dense("k", 0, h)[kept], old.dense("v", 0, h)[kept]
        for gq in range(group):
            s = k @ q[0, 0, h * group + gq].double().cpu().numpy() / math.sqrt(dim)
            p = np.exp(s - s.max())
            want = p @ v / p.sum()
            assert np.allclose(out[0, 0, h * group + gq].double().cpu().numpy(), want, rtol=2 ** -7, atol=2e-3)


def test_bounded_cache_refusals():
    from kvbridge_b200 import kv4_decode

    with pytest.raises(ValueError, match="budget"):
        kv4_decode.BoundedCache(1, 1, 64, 16, 100, 100, 0, 0, "cpu")
    with pytest.raises(ValueError, match="observe"):
        kv4_decode.decode(prompt=3, observe=4)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [
    dict(batch=3, prompt=700, steps=40, budget=200, slack=16, page_tokens=16, dim=64, q_heads=4, kv_heads=2),
    dict(batch=1, prompt=65, steps=70, budget=100, slack=1, page_tokens=32, dim=256, q_heads=6, kv_heads=1, observe=1),
    dict(batch=2, prompt=500, steps=20, budget=300, slack=300, page_tokens=64, q_heads=16, dtype=torch.float32),
])
def test_bounded_decode(cuda_device, kw):
    """The serving loop: how often it evicts, and its last output. Values are
    sums of normal numbers' 4-bit images with weights that add up to 1, so below
    6: bf16 rounds them to 6 * 2^-8, the 16-bit digits of P add 2^-15 of that."""
    from kvbridge_b200 import kv4_decode

    result = kv4_decode.decode(**kw, device=cuda_device)
    held, evictions, cap = kw["prompt"], 0, kw["budget"] + kw["slack"]
    for _ in range(kw["steps"]):
        if held >= cap:
            held, evictions = kw["budget"], evictions + 1
        held += 1
    assert (result["longest"], result["evictions"]) == (held, evictions)
    assert result["error"] < (2e-5 if kw.get("dtype") is torch.float32 else 6 * 2 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_append_codes_at_ties(cuda_device, dtype, dim):
    """Rows whose quotients lie at or next to half integers: codes are those of
    the rounded division, bit for bit."""
    g = torch.Generator().manual_seed(81)
    n, heads, page = 96, 2, 16
    half = torch.randint(0, 31, (n, heads, dim), generator=g).float() / 2  # 0, 0.5, .. 15
    half[..., 0], half[..., 1] = 0.0, 15.0
    x = half * torch.exp2(torch.randint(-20, 12, (n, heads, 1), generator=g).float())
    x = x * torch.where(torch.rand((n, heads, 1), generator=g) < 0.5, 1.0, 1.0 + 1.0 / 3)
    x = (x + torch.randn((n, heads, 1), generator=g) * (x.amax(-1, keepdim=True) / 8)).to(dtype)
    pool = kvb.Kv4Pool.empty(n // page, heads, page, dim, device=cuda_device)
    slots = torch.randperm(n, generator=g)
    kvb.append_kv4(pool, kvb.Kv4Rows(x.to(cuda_device), x.flip(0).contiguous().to(cuda_device), slots.to(cuda_device)))
    code, want = util.quantize(x.float())
    k = pool.k.cpu().transpose(1, 2).reshape(n, heads, dim // 2)[slots]
    assert torch.equal(k, util.pack(code))
    params = pool.k_params.cpu().transpose(1, 2).reshape(n, heads, 2)[slots]
    assert torch.equal(params, want)
    v = pool.v.cpu().permute(0, 3, 1, 2).reshape(n, heads, dim // 2)[slots]
    assert torch.equal(v.flip(0), util.pack(code))


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,group,dim", [(1, 8, 128), (1, 4, 256), (2, 1, 64)])
def test_attention_many_partials_a_row(cuda_device, kv_heads, group, dim):
    """Few long segments: as many partials a row as there can be."""
    cache = util.make_cache([9001, 33000], kv_heads, dim, 64, seed=91)
    rule = util.make_query(cache, util.Rule(rows=1, group=group, dtype=torch.float32), seed=92)
    util.check_attention(cache, rule, cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("rule", [dict(), dict(window=70), dict(window=40, prefix=[3] * 40, softcap=20.0)])
def test_attention_more_sequences_than_lanes(cuda_device, rule):
    lens = [(37 * b) % 301 for b in range(40)]
    cache = util.make_cache(lens, 2, 64, 16, seed=95)
    rule = util.make_query(cache, util.Rule(rows=2, group=3, **rule), seed=96)
    util.check_attention(cache, rule, cuda_device)
