"""Decoding over a 4-bit cache of bounded size, the operators of ``kv4``
together as a serving loop uses them: ``python -m kvbridge_b200.kv4_decode
--batch 4 --prompt 8000 --steps 200 --budget 2048``.

The prompt's K and V rows are appended, and the prompt's last query rows give
its tokens their first weights. Each step appends one token a sequence, attends
and adds up the attention weights. Where a sequence has ``budget + slack``
tokens, first every sequence keeps its ``budget`` (the first ``sinks``, the last
``recent`` and the heaviest of the rest) and moves to its other pages; tokens
keep their positions. Queries, keys and values are random numbers. Prints one
line: the time of a step, the evictions, and the last output's distance from a
softmax in 64 bits over what the cache holds.
"""
from __future__ import annotations

import argparse
import sys

import torch

import kvbridge_b200 as kvb


class BoundedCache:
    """A pool with two sets of pages a sequence, used in turn."""

    def __init__(self, batch, kv_heads, dim, page_tokens, capacity, budget, sinks, recent, device):
        if not 0 < budget < capacity:
            raise ValueError("budget must be positive and below the capacity")
        self.budget, self.sinks, self.recent, self.page_tokens = budget, sinks, recent, page_tokens
        self.capacity = capacity
        width = -(-capacity // page_tokens)
        self.pool = kvb.Kv4Pool.empty(2 * batch * width, kv_heads, page_tokens, dim, device, positions=True)
        pages = torch.randperm(2 * batch * width, device=device).int().view(2, batch, width)
        self.tables = [pages[0].contiguous(), pages[1].contiguous()]
        self.weights = [torch.zeros(batch, kv_heads, capacity, device=device) for _ in range(2)]
        self.keep = torch.empty(batch, kv_heads, budget, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.seen = torch.zeros(batch, dtype=torch.int32, device=device)  # tokens ever appended = the next position
        self.longest = 0  # of lens, on the host
        self.now = 0
        self.evictions = 0

    def slots(self, counts: torch.Tensor, tokens: int) -> torch.Tensor:
        """Slots of up to `tokens` tokens after each sequence's last (-1 beyond its count)."""
        step = torch.arange(tokens, device=counts.device)
        at = self.lens[:, None] + step
        page = (at // self.page_tokens).clamp(max=self.tables[0].shape[1] - 1)
        slot = self.tables[self.now].gather(1, page).long() * self.page_tokens + at % self.page_tokens
        return torch.where(step < counts[:, None], slot, -1)

    def append(self, k, v, counts=None) -> None:
        """K and V [batch, tokens, kv_heads, dim], the first counts[b] of each sequence."""
        batch, tokens = k.shape[:2]
        if self.longest + tokens > self.capacity:
            raise ValueError("the cache is full")
        if counts is None:
            counts = torch.full_like(self.lens, tokens)
        slots = self.slots(counts, tokens)
        positions = self.seen[:, None] + torch.arange(tokens, dtype=torch.int32, device=k.device)
        rows = kvb.Kv4Rows(k.flatten(0, 1), v.flatten(0, 1), slots.flatten(), positions.flatten())
        kvb.append_kv4(self.pool, rows)
        self.lens += counts
        self.seen += counts
        self.longest += tokens

    def query(self, q, scale) -> "kvb.Kv4Query":
        """Query rows [batch, rows, q_heads, dim] of the last tokens."""
        rows = q.shape[1]
        positions = self.seen[:, None] - rows + torch.arange(rows, dtype=torch.int32, device=q.device)
        return kvb.Kv4Query(q, self.lens, self.tables[self.now], self.longest, self.pool.kv_heads, scale,
                            q_positions=positions)

    def attend(self, q, scale):
        """Attention of the rows; their weights are added to the tokens'."""
        query = self.query(q, scale)
        space = torch.empty(kvb.attention_kv4_workspace_bytes(self.pool, query), dtype=torch.uint8, device=q.device)
        out, lse = torch.empty_like(q), torch.empty(q.shape[:3], device=q.device)
        kvb.launch_attention_kv4(self.pool, query, space, out, lse)
        kvb.accumulate_weights_kv4(self.pool, query, lse, self.weights[self.now])
        return out

    def evict(self) -> None:
        """Every sequence to at most the budget, on its other pages."""
        old, new = self.now, 1 - self.now
        plan = kvb.EvictPlan(self.weights[old], self.lens, self.tables[old], self.budget, self.sinks, self.recent)
        lens = torch.empty_like(self.lens)
        kvb.select_tokens(plan, self.keep, lens)
        self.weights[new].zero_()
        kvb.compact_kv4(self.pool, plan, self.keep, self.tables[new], self.weights[new])
        self.lens, self.now = lens, new
        self.longest = min(self.longest, self.budget)
        self.evictions += 1

    def contents(self, dtype=torch.float32):
        """What the cache holds: K, V [batch, longest, kv_heads, dim] and the
        positions [batch, kv_heads, longest] (past a sequence's end: anything)."""
        at = torch.arange(self.longest, device=self.lens.device).expand(self.lens.shape[0], -1)
        slots = self.tables[self.now].gather(1, at // self.page_tokens).long() * self.page_tokens + at % self.page_tokens
        shape = (slots.numel(), self.pool.kv_heads, self.pool.dim)
        k, v = torch.empty(shape, dtype=dtype, device=slots.device), torch.empty(shape, dtype=dtype, device=slots.device)
        slots = torch.where(at < self.lens[:, None], slots, -1)  # zeros past the end
        kvb.load_kv4(self.pool, kvb.Kv4Rows(k, v, slots.flatten()))
        flat = slots.clamp(min=0)
        positions = self.pool.positions[flat // self.page_tokens, :, flat % self.page_tokens].transpose(1, 2)
        return k.view(*slots.shape, *shape[1:]), v.view(*slots.shape, *shape[1:]), positions


def distance(cache: BoundedCache, q, scale, out) -> float:
    """Largest difference of `out` from a softmax in 64 bits over the cache's contents."""
    k, v, _ = cache.contents()
    group = q.shape[2] // cache.pool.kv_heads
    k, v = (x.double().repeat_interleave(group, dim=2) for x in (k, v))
    score = scale * torch.einsum("brhd,bthd->brht", q.double(), k)
    # One row, the last token's: it sees everything.
    past = torch.arange(k.shape[1], device=q.device) >= cache.lens[:, None]
    score.masked_fill_(past[:, None, None, :], float("-inf"))
    want = torch.einsum("brht,bthd->brhd", score.softmax(-1), v)
    return (want - out.double()).abs().max().item()


def decode(batch=4, prompt=8000, steps=200, budget=2048, slack=256, sinks=4, recent=64, q_heads=32, kv_heads=8,
           dim=128, page_tokens=64, observe=4, dtype=torch.bfloat16, seed=0, device="cuda") -> dict:
    if min(batch, steps, prompt, observe) < 1 or slack < 1 or observe > prompt:
        raise ValueError("batch, prompt, steps, slack and observe must be positive, observe at most the prompt")
    torch.manual_seed(seed)
    scale = dim**-0.5

    def rows(tokens, heads):
        return torch.randn(batch, tokens, heads, dim, device=device).to(dtype)

    # Ragged prompts, between half of `prompt` and all of it.
    counts = torch.randint((prompt + 1) // 2, prompt + 1, (batch,), device=device, dtype=torch.int32)
    counts[0] = prompt
    cache = BoundedCache(batch, kv_heads, dim, page_tokens, max(prompt, budget + slack), budget, sinks, recent, device)
    cache.append(rows(prompt, kv_heads), rows(prompt, kv_heads), counts)
    cache.attend(rows(observe, q_heads), scale)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(steps):
        if cache.longest >= budget + slack:
            cache.evict()
        cache.append(rows(1, kv_heads), rows(1, kv_heads))
        q = rows(1, q_heads)
        out = cache.attend(q, scale)
    end.record()
    end.synchronize()
    status = kvb.read_device_status()
    if status != 0:
        raise RuntimeError(f"device status {status}")
    return {
        "us_per_step": start.elapsed_time(end) / steps * 1e3,
        "evictions": cache.evictions,
        "longest": cache.longest,
        "error": distance(cache, q, scale, out),
    }


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, default in (("batch", 4), ("prompt", 8000), ("steps", 200), ("budget", 2048), ("slack", 256), ("sinks", 4),
                          ("recent", 64), ("q-heads", 32), ("kv-heads", 8), ("dim", 128), ("page-tokens", 64),
                          ("observe", 4), ("seed", 0)):
        ap.add_argument(f"--{name}", type=int, default=default)
    args = vars(ap.parse_args(argv))
    result = decode(**args)
    print("{us_per_step:.1f} us a step, {evictions} evictions, {longest} tokens held, largest error {error:.2e}".format(**result))
    return 0


if __name__ == "__main__":
    sys.exit(main())
