#pragma once
// Eviction from a cache by accumulated attention weight: the choice of the
// kept tokens, and their copy to new pages of the 4-bit pool.
#include <cooperative_groups.h>

#include "kv4_common.cuh"

namespace kvb {

namespace cg = cooperative_groups;

struct SelectParams {
  const uint32_t* seq_lens;
  const float* weights;
  int64_t weight_stride;
  int32_t* keep;
  uint32_t* kept_lens;
  uint32_t batch, kv_heads, max_tokens, budget, sinks, recent;
};

// Order-preserving image of a weight: larger weight, larger key; all NaNs
// alike and above +inf, -0 like +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 512;
constexpr uint32_t kSelectKeys = 16384;  // keys a CTA keeps in shared memory
constexpr uint32_t kSelectBins = 2048;   // four a thread

struct SelectSmem {
  uint32_t hist[2][kSelectBins];
  uint32_t prefix, want;
  uint32_t counts[2];  // of this CTA: kept without ties, ties
  uint32_t warp_sum[kSelectThreads / 32], warp_keep[kSelectThreads / 32], warp_tie[kSelectThreads / 32];
};

// One cluster per (sequence, KV head), a contiguous part of the tokens a CTA;
// the middle tokens' keys are read once and kept in shared memory (parts of
// more than kSelectKeys tokens are read again from L2). The budget - sinks -
// recent largest keys are found by their digits of 11, 11 and 10 bits, highest
// first: every CTA counts the keys that agree with the prefix so far, the CTAs
// add the counts up over distributed shared memory, and the digit is the one
// in which the count from the top reaches what is still wanted. (Eleven bits:
// weights share few exponents, and the counters of a byte were a queue.) Then
// one ordered pass: a token is kept if its key is above the threshold, or
// equal to it and among the first `want` of those. Bound by the chain of those
// steps, not by bytes (4 a token): 16 sequences of 1.5K to 16K tokens on 8
// heads 23 us, one of 128K on 2 heads about 28 us in clusters of eight.
__global__ void __launch_bounds__(kSelectThreads) select_tokens_kernel(SelectParams p) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ __align__(16) SelectSmem sm;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), ctas = cluster.num_blocks();
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t segment = blockIdx.x / ctas, b = segment / p.kv_heads;
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t len = kv4_len(p.seq_lens, b, p.max_tokens), kept = min(len, p.budget);
  if (tid == 0 && rank == 0 && segment % p.kv_heads == 0) {
    p.kept_lens[b] = kept;
    if (kv4_load(p.seq_lens + b) > p.max_tokens) atomicMax(&g_kvb_status, kKv4LenClamped);
  }
  int32_t* keep = p.keep + size_t(segment) * p.budget;
  for (uint32_t i = kept + rank * kSelectThreads + tid; i < p.budget; i += ctas * kSelectThreads) keep[i] = 0;
  if (len <= p.budget) {  // the same for the whole cluster
    for (uint32_t i = rank * kSelectThreads + tid; i < len; i += ctas * kSelectThreads) keep[i] = int32_t(i);
    return;
  }
  const float* weights = p.weights + int64_t(segment) * p.weight_stride;
  const uint32_t part = (len + ctas - 1) / ctas, from = min(rank * part, len), to = min(from + part, len);
  const uint32_t first = p.sinks, last = len - p.recent;  // the middle tokens
  const uint32_t lo = max(from, first), hi = max(min(to, last), lo);  // of this CTA
  const bool cached = part <= kSelectKeys;
  auto key_of = [&](uint32_t t) { return cached ? keys[t - from] : weight_key(kv4_load(weights + t)); };
  // A thread goes over tokens in a row; the odd count keeps a warp's reads of
  // the keys in different banks.
  const uint32_t run = ((part + kSelectThreads - 1) / kSelectThreads) | 1u;
  const uint32_t run_from = min(from + tid * run, to), run_to = min(run_from + run, to);
  const uint32_t run_lo = max(run_from, first), run_hi = max(min(run_to, last), run_lo);
  uint32_t prefix = 0, mask = 0, want = p.budget - p.sinks - p.recent;
  const bool any = want != 0;
  if (any) {
    if (cached) {
#pragma unroll 8
      for (uint32_t t = lo + tid; t < hi; t += kSelectThreads) keys[t - from] = weight_key(kv4_load(weights + t));
    }
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
      const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
      const uint32_t bins = round == 2 ? 1024 : kSelectBins;
      // Nobody reads this buffer any more: its readers, two rounds back, have
      // passed the last round's barrier.
      uint32_t* hist = sm.hist[round & 1];
      reinterpret_cast<uint4*>(hist)[tid] = make_uint4(0, 0, 0, 0);
      __syncthreads();
#pragma unroll 4
      for (uint32_t t = run_lo; t < run_hi; ++t) {
        const uint32_t key = key_of(t);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
      }
      cluster.sync();
      // This thread's four bins, from the top; CTAs of a cluster all add up the same.
      const uint32_t at = kSelectBins / 4 - 1 - tid;
      uint4 c = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (uint32_t r = 0; r < 8; ++r)
        if (r < ctas) {
          const uint4 x = reinterpret_cast<const uint4*>(cluster.map_shared_rank(hist, r))[at];
          c.x += x.x, c.y += x.y, c.z += x.z, c.w += x.w;
        }
      const uint32_t own = c.x + c.y + c.z + c.w;
      uint32_t upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= uint32_t(o)) upto += y;
      }
      if (lane == 31) sm.warp_sum[warp] = upto;
      __syncthreads();
      upto += __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_sum[lane] : 0u);
      uint32_t above = upto - own;  // keys in higher bins
      if (above < want && upto >= want) {
        uint32_t bin = 4 * at + 3;
        if (above + c.w < want) {
          above += c.w, --bin;
          if (above + c.z < want) {
            above += c.z, --bin;
            if (above + c.y < want) above += c.y, --bin;
          }
        }
        sm.prefix = prefix | bin << shift;
        sm.want = want - above;
      }
      __syncthreads();
      prefix = sm.prefix;
      want = sm.want;
      mask |= (bins - 1) << shift;
    }
  }
  // `want` tokens whose key equals `prefix` are kept, the lowest first.
  uint32_t mine = 0, ties = 0;
  for (uint32_t t = run_from; t < run_to; ++t) {
    if (t < first || t >= last) {
      ++mine;
    } else if (any) {
      const uint32_t key = key_of(t);
      mine += key > prefix;
      ties += key == prefix;
    }
  }
  // Sums over the threads before this one, then over the CTAs before this one.
  uint32_t keep_upto = mine, tie_upto = ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, keep_upto, o), y = __shfl_up_sync(0xffffffffu, tie_upto, o);
    if (lane >= uint32_t(o)) keep_upto += x, tie_upto += y;
  }
  if (lane == 31) sm.warp_keep[warp] = keep_upto, sm.warp_tie[warp] = tie_upto;
  __syncthreads();
  const bool holds = lane < kSelectThreads / 32;
  const uint32_t warp_keep = holds ? sm.warp_keep[lane] : 0u, warp_tie = holds ? sm.warp_tie[lane] : 0u;
  uint32_t out = keep_upto - mine + __reduce_add_sync(0xffffffffu, lane < warp ? warp_keep : 0u);
  uint32_t seen = tie_upto - ties + __reduce_add_sync(0xffffffffu, lane < warp ? warp_tie : 0u);
  const uint32_t all_keep = __reduce_add_sync(0xffffffffu, warp_keep), all_tie = __reduce_add_sync(0xffffffffu, warp_tie);
  if (tid == 0) sm.counts[0] = all_keep, sm.counts[1] = all_tie;
  cluster.sync();
  for (uint32_t r = 0; r < rank; ++r) {
    const uint32_t* counts = cluster.map_shared_rank(sm.counts, r);
    out += counts[0];
    seen += counts[1];
  }
  cluster.sync();  // the counts are read: CTAs may leave
  out += min(seen, want);
  for (uint32_t t = run_from; t < run_to; ++t) {
    bool take = t < first || t >= last;
    if (!take && any) {
      const uint32_t key = key_of(t);
      take = key > prefix || (key == prefix && seen++ < want);
    }
    if (take) keep[out++] = int32_t(t);
  }
}

struct CompactParams {
  Kv4View pool;
  const uint32_t* seq_lens;
  const float* weights;
  int64_t weight_stride;
  const uint32_t* table;
  const int32_t* keep;
  const uint32_t* new_table;
  float* new_weights;
  int64_t new_weight_stride;
  uint32_t batch, max_tokens, budget, table_stride, new_stride, page_tokens, log2_page;
};

constexpr int kCompactThreads = 256;
constexpr uint32_t kCompactTile = 64;  // kept tokens a CTA
// Bytes of source V pages held at once, and gaps: two of the largest pages. Eight
// CTAs fit an SM (twice the bytes and five CTAs: 16 sequences of up to 16K tokens
// selected and moved in 82 us, with this in 75; half of it is no faster).
constexpr uint32_t kCompactStage = 16384 + 512;

// One CTA per (64 kept tokens, KV head, sequence). A kept token's V bytes lie
// in every sector row of its page, so that V costs whole source pages: 143 MB
// read where 16 sequences of up to 16K tokens on 8 heads keep 2,048 (38 MB), 49
// us. Bound by the latency of its steps in a row (token list, table, pages,
// picking, stores) at eight CTAs an SM, whose waits do not overlap enough to
// fill the HBM. K rows and params go straight across. V pages come in whole
// (16-byte copies) into shared memory, the kept tokens' bytes are picked into a
// tile of the new layout, and the tile is stored in 16-byte runs. Slots after
// the kept ones are not written.
template <int D>
__global__ void __launch_bounds__(kCompactThreads) compact_kv4_kernel(const CompactParams p) {
  __shared__ __align__(16) uint8_t stage[kCompactStage];
  __shared__ __align__(16) uint8_t tile[D / 2][kCompactTile];
  __shared__ uint64_t src_at[kCompactTile], dst_unit[4];  // element of the params; units of the new pages
  __shared__ uint64_t run_src[kCompactTile];              // source pages, a run of tokens each: where their V lies
  __shared__ uint32_t src_slot[kCompactTile], order[kCompactTile], page_of[kCompactTile];
  __shared__ uint32_t runs_sh;
  constexpr uint64_t kNowhere = ~uint64_t(0);
  const uint32_t tid = threadIdx.x, h = blockIdx.y, b = blockIdx.z, H = p.pool.kv_heads;
  const uint32_t P = p.page_tokens, first = blockIdx.x * kCompactTile;
  grid_launch_dependents();
  grid_dependency_wait();
  const uint32_t len = kv4_len(p.seq_lens, b, p.max_tokens), kept = min(len, p.budget);
  if (first == 0 && h == 0 && tid == 0 && kv4_load(p.seq_lens + b) > p.max_tokens) atomicMax(&g_kvb_status, kKv4LenClamped);
  const size_t row = size_t(b) * H + h;
  const int32_t* keep = p.keep + row * p.budget;
  if (tid < 64) {  // two whole warps
    const uint32_t i = first + tid;
    uint64_t at = kNowhere;
    uint32_t page = 0xffffffffu, slot = 0;
    float weight = 0.f;
    if (i < kept) {
      const uint32_t t = uint32_t(kv4_load(keep + i));
      if (t < len && (t >> p.log2_page) < p.table_stride) {
        weight = kv4_load(p.weights + int64_t(row) * p.weight_stride + t);
        page = kv4_load(p.table + size_t(b) * p.table_stride + (t >> p.log2_page));
        slot = t & (P - 1);
        if (page < p.pool.pages)
          at = (uint64_t(page) * H + h) * P + slot;
        else
          atomicMax(&g_kvb_status, kKv4BadPage);
      } else {
        atomicMax(&g_kvb_status, kKv4BadKept);
      }
    }
    if (p.new_weights != nullptr && i < p.budget) p.new_weights[int64_t(row) * p.new_weight_stride + i] = weight;
    src_at[tid] = at;
    src_slot[tid] = slot;
    page_of[tid] = at != kNowhere ? page : 0xffffffffu;
  }
  if (tid < 4) {
    const uint32_t j = (first + 16 * tid) >> p.log2_page;
    uint64_t unit = kNowhere;
    if (first + 16 * tid < kept) {
      const uint32_t page = kv4_load(p.new_table + size_t(b) * p.new_stride + j);
      if (page < p.pool.pages)
        unit = uint64_t(page) * H + h;
      else
        atomicMax(&g_kvb_status, kKv4BadPage);
    }
    dst_unit[tid] = unit;  // of the page of tokens 16 tid ..
  }
  __syncthreads();
  if (first >= kept) return;
  // Number the runs of tokens of one source page.
  if (tid < 32) {
    uint32_t before = 0;
#pragma unroll
    for (uint32_t base = 0; base < kCompactTile; base += 32) {
      const uint32_t i = base + tid;
      const bool starts = i == 0 || page_of[i] != page_of[i - 1];
      const uint32_t mask = __ballot_sync(0xffffffffu, starts);
      const uint32_t run = before + __popc(mask & (0xffffffffu >> (31 - tid))) - 1;
      order[i] = run;
      if (starts) run_src[run] = src_at[i] == kNowhere ? kNowhere : (src_at[i] - src_slot[i]) * (D / 2);
      before += __popc(mask);
    }
    if (tid == 0) runs_sh = before;
  }
  __syncthreads();
  // V, as many source pages at a time as the stage holds, 16 bytes apart: a
  // page's 16-byte chunks by neighbouring threads.
  const uint32_t page_bytes = P * (D / 2), pitch = page_bytes + 16;
  const uint32_t log2_chunks = p.log2_page + (D == 64 ? 1 : D == 128 ? 2 : 3);
  const uint32_t runs = runs_sh, together = min(kCompactStage / pitch, kCompactTile);
  auto fetch = [&](uint32_t base) {
    const uint32_t here = min(together, runs - base) << log2_chunks;
#pragma unroll 4
    for (uint32_t i = tid; i < here; i += kCompactThreads) {
      const uint32_t r = i >> log2_chunks, c = i & ((1u << log2_chunks) - 1);
      const uint64_t src = run_src[base + r];
      if (src != kNowhere) copy16_async(smem_addr(stage) + r * pitch + 16 * c, p.pool.v + src + 16 * c);
    }
    copy_commit();
  };
  fetch(0);
  // K rows, params and positions meanwhile.
  constexpr uint32_t kChunks = D / 32;  // 16-byte chunks of a K row
#pragma unroll
  for (uint32_t i = tid; i < kCompactTile * kChunks; i += kCompactThreads) {
    const uint32_t t = i / kChunks, c = i % kChunks;
    const uint64_t from = src_at[t], unit = dst_unit[t / 16];
    if (unit == kNowhere || first + t >= kept) continue;
    const uint64_t to = unit * P + ((first + t) & (P - 1));
    if (from == kNowhere) {  // a row that is not a number, for whatever the slot holds
      if (c < 2) {
        const float nan = __int_as_float(0x7fffffff);
        (c == 0 ? p.pool.kp : p.pool.vp)[to] = make_float2(nan, nan);
        if (c == 0 && p.pool.pos != nullptr) p.pool.pos[to] = 0;
      }
      continue;
    }
    reinterpret_cast<uint4*>(p.pool.k)[to * kChunks + c] = kv4_stream(reinterpret_cast<const uint4*>(p.pool.k) + from * kChunks + c);
    if (c == 0) p.pool.kp[to] = p.pool.kp[from];
    if (c == 1) p.pool.vp[to] = p.pool.vp[from];
    if (c == kChunks - 1 && p.pool.pos != nullptr) p.pool.pos[to] = p.pool.pos[from];
  }
  for (uint32_t base = 0; base < runs; base += together) {
    if (base != 0) {
      __syncthreads();  // the stage has been read
      fetch(base);
    }
    copy_wait<0>();
    __syncthreads();
    // A warp takes 32 tokens of a dim pair.
    const uint32_t t = tid % kCompactTile;
    if (order[t] >= base && order[t] < base + together && src_at[t] != kNowhere) {
      const uint8_t* src = stage + (order[t] - base) * pitch + src_slot[t];
#pragma unroll 8
      for (uint32_t c = tid / kCompactTile; c < D / 2; c += kCompactThreads / kCompactTile) tile[c][t] = src[c * P];
    }
  }
  __syncthreads();
  for (uint32_t i = tid; i < 4 * (D / 2); i += kCompactThreads) {
    const uint32_t g = i % 4, c = i / 4, t = 16 * g;  // 16 tokens of a dim pair
    if (dst_unit[g] == kNowhere) continue;
    uint8_t* dst = p.pool.v + (dst_unit[g] * (D / 2) + c) * P + ((first + t) & (P - 1));
    bool whole = true;
    for (uint32_t k = 0; k < 16; ++k) whole = whole && src_at[t + k] != kNowhere;
    if (whole) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(&tile[c][t]);
    } else {
      for (uint32_t k = 0; k < 16; ++k)
        if (src_at[t + k] != kNowhere) dst[k] = tile[c][t + k];
    }
  }
}

}  // namespace kvb
