#pragma once
// Eviction from a cache by accumulated attention weight: the choice of the
// kept tokens, and their copy to new pages of the 4-bit pool.
#include "kv4_common.cuh"

namespace kvb {

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

constexpr int kSelectThreads = 1024;

// One CTA per (sequence, KV head). The budget - sinks - recent largest keys
// of the middle tokens are found by their bytes, highest first: a histogram
// of the keys that agree with the prefix so far, then the byte in which the
// count from the top reaches what is still wanted. Then one ordered pass:
// a token is kept if its key is above the threshold, or equal to it and
// among the first `ties` of those.
__global__ void __launch_bounds__(kSelectThreads) select_tokens_kernel(SelectParams p) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sh_prefix, sh_want;
  __shared__ uint32_t scan_keep[32], scan_tie[32];
  grid_dependency_wait();
  const uint32_t tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const uint32_t b = blockIdx.x / p.kv_heads, h = blockIdx.x % p.kv_heads;
  const uint32_t len = kv4_len(p.seq_lens, b, p.max_tokens);
  const uint32_t kept = min(len, p.budget);
  if (tid == 0 && h == 0) {
    p.kept_lens[b] = kept;
    if (__ldg(p.seq_lens + b) > p.max_tokens) atomicMax(&g_kvb_status, kKv4LenClamped);
  }
  int32_t* keep = p.keep + size_t(blockIdx.x) * p.budget;
  for (uint32_t i = kept + tid; i < p.budget; i += kSelectThreads) keep[i] = 0;
  if (len <= p.budget) {
    for (uint32_t i = tid; i < len; i += kSelectThreads) keep[i] = int32_t(i);
    return;
  }
  const float* weights = p.weights + int64_t(blockIdx.x) * p.weight_stride;
  const uint32_t first = p.sinks, last = len - p.recent;  // the middle tokens
  uint32_t prefix = 0, mask = 0, want = p.budget - p.sinks - p.recent;
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (uint32_t t = first + tid; t < last; t += kSelectThreads) {
      const uint32_t key = weight_key(weights[t]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = want;
      int d = 255;
      for (; d > 0 && hist[d] < left; --d) left -= hist[d];
      sh_prefix = prefix | (uint32_t(d) << shift);
      sh_want = left;
    }
    __syncthreads();
    prefix = sh_prefix;
    want = sh_want;
    mask |= 255u << shift;
    __syncthreads();
  }
  // `want` of the tokens whose key equals `prefix` are kept, the lowest first
  // (none when nothing of the middle is wanted).
  const bool any = p.budget > p.sinks + p.recent;
  uint32_t out = 0, ties = 0;
  for (uint32_t base = 0; base < len; base += kSelectThreads) {
    const uint32_t t = base + tid;
    bool take = false, tie = false;
    if (t < len) {
      if (t < first || t >= last) {
        take = true;
      } else if (any) {
        const uint32_t key = weight_key(weights[t]);
        take = key > prefix;
        tie = key == prefix;
      }
    }
    const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) scan_tie[w] = __popc(tie_mask);
    __syncthreads();
    uint32_t tie_rank = ties + __popc(tie_mask & ((1u << lane) - 1u)), tie_all = 0;
    for (uint32_t i = 0; i < 32; ++i) {
      if (i < w) tie_rank += scan_tie[i];
      tie_all += scan_tie[i];
    }
    take = take || (tie && tie_rank < want);
    const uint32_t keep_mask = __ballot_sync(0xffffffffu, take);
    if (lane == 0) scan_keep[w] = __popc(keep_mask);
    __syncthreads();
    uint32_t at = out + __popc(keep_mask & ((1u << lane) - 1u)), all = 0;
    for (uint32_t i = 0; i < 32; ++i) {
      if (i < w) at += scan_keep[i];
      all += scan_keep[i];
    }
    if (take) keep[at] = int32_t(t);
    out += all;
    ties += tie_all;
    __syncthreads();
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
  uint32_t batch, max_tokens, budget, table_stride, new_stride;
};

// One CTA of 128 threads per (new page, KV head, sequence).
template <int D>
__global__ void __launch_bounds__(128) compact_kv4_kernel(CompactParams p, uint32_t P) {
  grid_dependency_wait();
  const uint32_t tid = threadIdx.x, j = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const uint32_t H = p.pool.kv_heads;
  const uint32_t len = kv4_len(p.seq_lens, b, p.max_tokens);
  if (j == 0 && h == 0 && tid == 0 && __ldg(p.seq_lens + b) > p.max_tokens)
    atomicMax(&g_kvb_status, kKv4LenClamped);
  const uint32_t kept = min(len, p.budget);
  const int32_t* keep = p.keep + (size_t(b) * H + h) * p.budget;
  const uint32_t end = min(p.budget, (j + 1) * P);
  if (p.new_weights != nullptr)
    for (uint32_t i = j * P + tid; i < end; i += 128) {
      const uint32_t t = uint32_t(keep[i]);
      const bool ok = i < kept && t < len;
      p.new_weights[(int64_t(b) * H + h) * p.new_weight_stride + i] =
          ok ? p.weights[(int64_t(b) * H + h) * p.weight_stride + t] : 0.f;
    }
  if (j * P >= kept) return;
  const uint32_t to = p.new_table[size_t(b) * p.new_stride + j];
  if (to >= p.pool.pages) {
    if (tid == 0) atomicMax(&g_kvb_status, kKv4BadPage);
    return;
  }
  const uint64_t dst = uint64_t(to) * H + h;
  for (uint32_t i = j * P; i < min(end, kept); ++i) {
    const uint32_t t = uint32_t(keep[i]);
    if (t >= len || t / P >= p.table_stride) {
      if (tid == 0) atomicMax(&g_kvb_status, kKv4BadKept);
      continue;
    }
    const uint32_t from = p.table[size_t(b) * p.table_stride + t / P], s = t % P, d = i % P;
    if (from >= p.pool.pages) {
      if (tid == 0) atomicMax(&g_kvb_status, kKv4BadPage);
      continue;
    }
    const uint64_t src = uint64_t(from) * H + h;
    for (uint32_t c = tid; c < D / 2; c += 128) {
      p.pool.k[(dst * P + d) * (D / 2) + c] = p.pool.k[(src * P + s) * (D / 2) + c];
      p.pool.v[(dst * (D / 2) + c) * P + d] = p.pool.v[(src * (D / 2) + c) * P + s];
    }
    if (tid == 0) {
      p.pool.kp[dst * P + d] = p.pool.kp[src * P + s];
      p.pool.vp[dst * P + d] = p.pool.vp[src * P + s];
      if (p.pool.pos != nullptr) p.pool.pos[dst * P + d] = p.pool.pos[src * P + s];
    }
  }
}

}  // namespace kvb
