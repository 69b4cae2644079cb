"""Plain 64-bit restatement of the 4-bit cache operators, and inputs for them."""
from __future__ import annotations

import math
from dataclasses import dataclass, field, replace
from typing import Optional

import numpy as np
import torch

EPS = 2.0 ** -24  # half an fp32 ulp, relative


def quantize(x: torch.Tensor):
    """Codes [.., dim] (uint8) and params [.., 2] of fp32 rows, in fp32 as the format says."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = (hi - lo) * (torch.tensor(1.0) / torch.tensor(15.0))
    ok = torch.isfinite(x).all(-1, keepdim=True) & torch.isfinite(scale)
    code = ((x - lo) / torch.where(scale > 0, scale, torch.ones_like(scale))).round().clamp(0, 15)
    code = torch.where(ok, code, torch.zeros_like(code)).to(torch.uint8)
    return code, torch.where(ok, torch.cat([scale, lo], -1), torch.nan)


def pack(code: torch.Tensor) -> torch.Tensor:
    return code[..., 0::2] | (code[..., 1::2] << 4)


@dataclass
class Cache:
    """A CPU pool with its dense 64-bit values beside it."""

    k: torch.Tensor
    v: torch.Tensor
    k_params: torch.Tensor
    v_params: torch.Tensor
    table: torch.Tensor  # int32 [batch, width]
    lens: list
    page: int
    positions: Optional[torch.Tensor] = None

    @property
    def heads(self):
        return self.k.shape[1]

    @property
    def dim(self):
        return 2 * self.k.shape[3]

    def dense(self, what: str, b: int, h: int) -> np.ndarray:
        """Values [len, dim] of one sequence and head."""
        n = self.lens[b]
        t = np.arange(n)
        pages, s = self.table[b].numpy()[t // self.page].astype(np.int64), t % self.page
        if what == "k":
            byte, par = self.k.numpy()[pages, h, s], self.k_params.numpy()[pages, h, s]
        else:
            byte, par = self.v.numpy()[pages, h, :, s], self.v_params.numpy()[pages, h, s]
        code = np.empty((n, self.dim))
        code[:, 0::2], code[:, 1::2] = byte & 15, byte >> 4
        par = par.astype(np.float64)
        return par[:, 1:] + par[:, :1] * code

    def token_positions(self, b: int, h: int) -> np.ndarray:
        t = np.arange(self.lens[b])
        if self.positions is None:
            return t
        return self.positions.numpy()[self.table[b].numpy()[t // self.page].astype(np.int64), h, t % self.page].astype(np.int64)

    def to(self, device):
        import kvbridge_b200 as kvb

        pos = None if self.positions is None else self.positions.to(device)
        return kvb.Kv4Pool(*(x.to(device) for x in (self.k, self.v, self.k_params, self.v_params)), positions=pos)


def make_cache(lens, heads, dim, page, seed, spare=2, positions=False, garbage=True) -> Cache:
    """Filled pages in shuffled order. Slots past a sequence's end hold random
    codes and, with `garbage`, NaN and infinite params."""
    g = torch.Generator().manual_seed(seed)
    each = [-(-n // page) for n in lens]
    pages = sum(each) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = max(1, max(each))
    table = torch.full((len(lens), width), 0, dtype=torch.int32)
    shape = (pages, heads, page)
    k = torch.randn(shape + (dim,), generator=g) + torch.randn((heads, 1, dim), generator=g)
    v = torch.randn(shape + (dim,), generator=g)
    v *= 1 + 9 * (torch.rand(shape + (1,), generator=g) < 0.05)
    kc, kp = quantize(k)
    vc, vp = quantize(v)
    used = torch.zeros((pages, page), dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        table[b, :each[b]] = order[at:at + each[b]]
        for j in range(each[b]):
            used[order[at + j], :min(page, n - j * page)] = True
        at += each[b]
    if garbage:
        kp[~used.unsqueeze(1).expand(shape)] = math.nan
        vp[~used.unsqueeze(1).expand(shape)] = math.inf
    pos = None
    if positions:
        pos = torch.full(shape, 1 << 30, dtype=torch.int32)
        for b, n in enumerate(lens):
            steps = torch.randint(1, 4, (heads, n), generator=g).cumsum(-1).to(torch.int32)
            for t in range(n):
                pos[table[b, t // page], :, t % page] = steps[:, t]
    return Cache(pack(kc), pack(vc).transpose(-1, -2).contiguous(), kp, vp, table, list(lens), page, pos)


@dataclass
class Rule:
    rows: int = 1
    group: int = 4
    softcap: float = 0.0
    slopes: bool = False
    window: int = 0
    prefix: Optional[list] = None
    dtype: torch.dtype = torch.float16
    q: torch.Tensor = field(default=None)
    q_positions: Optional[torch.Tensor] = None

    def slope_values(self, heads):
        n = heads * self.group
        return torch.exp2(-8.0 * (torch.arange(n) + 1) / n)


def make_query(cache: Cache, rule: Rule, seed: int) -> Rule:
    rule = replace(rule)
    g = torch.Generator().manual_seed(seed)
    shape = (len(cache.lens), rule.rows, cache.heads * rule.group, cache.dim)
    rule.q = (1.5 * torch.randn(shape, generator=g)).to(rule.dtype)
    if cache.positions is not None:
        last = [max((int(cache.token_positions(b, h).max(initial=-1)) for h in range(cache.heads)), default=-1)
                for b in range(len(cache.lens))]
        rule.q_positions = torch.tensor([[p + 1 + r for r in range(rule.rows)] for p in last], dtype=torch.int32)
    return rule


def device_query(cache: Cache, rule: Rule, device, max_tokens=None, strided=False):
    import kvbridge_b200 as kvb

    q = rule.q.to(device)
    if strided:  # columns of a wider projection
        wide = torch.randn(q.shape[:2] + (q.shape[2] + 3, q.shape[3]), device=device).to(q.dtype)
        wide[:, :, 1:1 + q.shape[2]] = q
        q = wide[:, :, 1:1 + q.shape[2]]
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return kvb.Kv4Query(
        q, as_int(cache.lens), cache.table.to(device),
        max_tokens=max(cache.lens) if max_tokens is None else max_tokens, kv_heads=cache.heads,
        scale=1 / math.sqrt(cache.dim), softcap=rule.softcap,
        slopes=rule.slope_values(cache.heads).to(device) if rule.slopes else None, window=rule.window,
        prefix_lens=None if rule.prefix is None else as_int(rule.prefix),
        q_positions=None if rule.q_positions is None else rule.q_positions.to(device))


@dataclass
class Expected:
    out: np.ndarray  # [batch, rows, q_heads, dim]
    lse: np.ndarray  # [batch, rows, q_heads]
    weights: list  # per sequence [heads, len]: weight of each token in this step
    out_tol: np.ndarray  # like out
    lse_tol: np.ndarray
    weight_tol: list


ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def expected(cache: Cache, rule: Rule) -> Expected:
    """The operators in 64 bits, with the error that the formats of the
    intermediate values allow:

    * scores: a query value is held to 2^-16 of its row's largest for 16-bit
      queries (2^-23 for fp32 ones and for the weights), so a score is off by
      that times scale * max|q| * sum|x|; the fp32 fold of the two terms scale_t *
      (q . code) and lo * sum q costs a few 2^-24 of scale * (|lo| + 15 scale_t) *
      sum|q|, the cap 2^-21 of softcap, the bias 2^-23 of itself.
    * attention weights: twice the score's error, and 2^-20 for exp and its sum.
    * probabilities times v scales are held to 2^-16 (fp32: 2^-22) of the
      largest of a tile, so each of n tokens adds up to 15 scale times that.
    * the result's own rounding.
    """
    B, R, G, H, D = len(cache.lens), rule.rows, rule.group, cache.heads, cache.dim
    scale = 1 / math.sqrt(D)
    out, lse = np.zeros((B, R, H * G, D)), np.full((B, R, H * G), -math.inf)
    out_tol, lse_tol = np.zeros_like(out), np.zeros_like(lse)
    weights, weight_tol = [], []
    fine = rule.dtype == torch.float32
    slopes = rule.slope_values(H).double().numpy()
    for b, n in enumerate(cache.lens):
        w, wt = np.zeros((H, n)), np.zeros((H, n))
        for h in range(H):
            k, v = cache.dense("k", b, h), cache.dense("v", b, h)
            pk = cache.token_positions(b, h)
            vpar = v.max(-1, initial=0) - v.min(-1, initial=0) if n else np.zeros(0)
            for r in range(R):
                pq = n - R + r if cache.positions is None else int(rule.q_positions[b, r])
                see = (pk <= pq) & ((pq - pk < rule.window) if rule.window else True)
                if rule.prefix is not None:
                    see |= pk < rule.prefix[b]
                if not see.any():
                    continue
                for gq in range(G):
                    head = h * G + gq
                    q = rule.q[b, r, head].double().numpy()
                    with np.errstate(invalid="ignore"):
                        x = scale * (k[see] @ q)
                        mag = scale * np.abs(q).sum() * np.abs(k[see]).max(initial=0)
                        grid = scale * np.abs(q).max() * np.abs(k[see]).sum(-1).max(initial=0)
                    fold = 16 * EPS * mag
                    err = {True: grid * 2.0 ** -23 + fold, False: grid * 2.0 ** -16 + fold}
                    extra = 8 * EPS * np.abs(x).max()
                    if rule.softcap:
                        x = rule.softcap * np.tanh(x / rule.softcap)
                        extra += 16 * EPS * rule.softcap
                    if rule.slopes:
                        bias = slopes[head] * np.abs(pq - pk[see])
                        x = x - bias
                        # far tokens carry no weight: what matters is the bias of those within 40 of the top
                        near = x > x.max() - 40
                        extra += 8 * EPS * (np.abs(bias[near]).max() + np.abs(x[near]).max())
                    top = x.max()
                    e = np.exp(x - top)
                    total = e.sum()
                    p = e / total
                    out[b, r, head] = p @ v[see]
                    lse[b, r, head] = top + math.log(total)
                    score = err[fine] + extra
                    lse_tol[b, r, head] = score + 2.0 ** -20 + 4 * EPS * abs(lse[b, r, head])
                    rel = 2 * score + 2.0 ** -20
                    grain = 2.0 ** (-22 if fine else -16)
                    spread = len(p) * p.max() * vpar[see].max()
                    out_tol[b, r, head] = (rel * np.abs(v[see]).max() + grain * spread
                                           + ROUND[rule.dtype] * np.abs(out[b, r, head]) + SMALLEST[rule.dtype])
                    w[h, see] += p
                    wt[h, see] += p * (2 * (err[True] + extra) + 2.0 ** -19 + 2 * lse_tol[b, r, head])
        weights.append(w)
        weight_tol.append(wt)
    return Expected(out, lse, weights, out_tol, lse_tol, weight_tol)


def attend(cache: Cache, rule: Rule, device, pool=None, query=None, **kw):
    """(out, lse) of the library, on the CPU in 64 bits."""
    import kvbridge_b200 as kvb

    pool = cache.to(device) if pool is None else pool
    query = device_query(cache, rule, device, **kw) if query is None else query
    ws = torch.full((kvb.attention_kv4_workspace_bytes(pool, query),), 0xFF, dtype=torch.uint8, device=device)
    out = torch.full(query.shape, math.nan, dtype=rule.dtype, device=device)
    lse = torch.full(query.shape[:3], math.nan, device=device)
    kvb.launch_attention_kv4(pool, query, ws, out, lse)
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), lse.double().cpu().numpy()


def check_attention(cache, rule, device, **kw):
    want = expected(cache, rule)
    out, lse = attend(cache, rule, device, **kw)
    empty = np.isneginf(want.lse)
    assert np.array_equal(empty, np.isneginf(lse))
    assert np.all(out[empty] == 0)
    off = np.abs(lse[~empty] - want.lse[~empty])
    assert np.all(off <= want.lse_tol[~empty]), (off.max(), want.lse_tol[~empty].min())
    off = np.abs(out - want.out)
    assert np.all(off <= want.out_tol), (off.max(), (off / np.maximum(want.out_tol, 1e-30)).max())
    return out, lse
