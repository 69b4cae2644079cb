#pragma once
// Attention over the 4-bit pool, and the attention weight that each cached
// token gets.
#include "kv4_common.cuh"

namespace kvb {

struct Kv4AttendParams {
  Kv4View pool;
  Kv4Rule rule;
  const void* q;
  int64_t batch_stride, row_stride;
  const uint32_t* seq_lens;
  const uint32_t* table;
  uint32_t batch, rows, q_heads, group, table_stride, max_tokens;
  void* out;
  float* lse;
  // accumulate_weights_kv4
  const float* lse_in;
  float* weights;
  int64_t weight_stride;
};

// Score of one token for one query row held in shared memory, or -inf.
template <int D>
__device__ float kv4_score(const Kv4AttendParams& p, const float* q, uint32_t P, uint64_t unit,
                           uint32_t s, int32_t pk, int32_t pq, float slope, uint32_t prefix) {
  if (!kv4_visible(pk, pq, p.rule.window, prefix)) return -INFINITY;
  const uint8_t* row = p.pool.k + (unit * P + s) * (D / 2);
  float dot = 0.f, sum = 0.f;
  for (int i = 0; i < D / 2; ++i) {
    const uint32_t b = row[i];
    dot = fmaf(q[2 * i], float(b & 15u), dot);
    dot = fmaf(q[2 * i + 1], float(b >> 4), dot);
    sum += q[2 * i] + q[2 * i + 1];
  }
  const float2 par = p.pool.kp[unit * P + s];
  float x = p.rule.scale * fmaf(par.x, dot, par.y * sum);
  if (p.rule.softcap > 0.f) x = p.rule.softcap * tanhf(x / p.rule.softcap);
  return x - slope * fabsf(float(pq - pk));
}

// One CTA of D threads per (sequence, query row, query head): tiles of D
// tokens, one score a thread, then one output dim a thread.
template <class T, int D>
__global__ void __launch_bounds__(D) attend_kv4_rows_kernel(Kv4AttendParams p, uint32_t P) {
  __shared__ float q[D], ps[D], pl[D], red[D / 32];
  __shared__ const uint8_t* vat[D];
  grid_dependency_wait();
  const uint32_t tid = threadIdx.x;
  const uint32_t head = blockIdx.x % p.q_heads, br = blockIdx.x / p.q_heads;
  const uint32_t r = br % p.rows, b = br / p.rows, h = head / p.group;
  const uint32_t len = kv4_len(p.seq_lens, b, p.max_tokens);
  if (tid == 0 && __ldg(p.seq_lens + b) > p.max_tokens) atomicMax(&g_kvb_status, kKv4LenClamped);
  q[tid] = to_f32(static_cast<const T*>(p.q)[int64_t(b) * p.batch_stride + int64_t(r) * p.row_stride + head * D + tid]);
  const int32_t pq = kv4_query_position(p.rule, b, r, p.rows, len);
  const float slope = p.rule.slopes != nullptr ? p.rule.slopes[head] : 0.f;
  const uint32_t prefix = p.rule.prefix != nullptr ? p.rule.prefix[b] : 0u;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (uint32_t base = 0; base < len; base += D) {
    const uint32_t t = base + tid;
    float x = -INFINITY;
    uint64_t unit = 0;
    uint32_t s = 0;
    __syncthreads();
    if (t < len) {
      const uint32_t page = p.table[size_t(b) * p.table_stride + t / P];
      s = t % P;
      if (page < p.pool.pages) {
        unit = uint64_t(page) * p.pool.kv_heads + h;
        const int32_t pk = p.pool.pos != nullptr ? p.pool.pos[unit * P + s] : int32_t(t);
        x = kv4_score<D>(p, q, P, unit, s, pk, pq, slope, prefix);
      } else {
        atomicMax(&g_kvb_status, kKv4BadPage);
      }
    }
    float mx = warp_max(x);
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    for (int i = 0; i < D / 32; ++i) mx = fmaxf(mx, red[i]);
    const float mnew = fmaxf(m, mx);
    const float base_m = mnew == -INFINITY ? 0.f : mnew;
    const float alpha = m == -INFINITY ? 0.f : expf(m - base_m);
    const bool on = x != -INFINITY;
    const float e = on ? expf(x - base_m) : 0.f;
    const float2 par = on ? p.pool.vp[unit * P + s] : make_float2(0.f, 0.f);
    ps[tid] = on ? e * par.x : 0.f;
    pl[tid] = on ? e * par.y : 0.f;
    vat[tid] = on ? p.pool.v + unit * (D / 2) * P + s : nullptr;
    const float sum = warp_sum(e);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = sum;
    __syncthreads();
    float lsum = 0.f;
    for (int i = 0; i < D / 32; ++i) lsum += red[i];
    l = l * alpha + lsum;
    acc *= alpha;
    for (int i = 0; i < D; ++i)
      if (vat[i] != nullptr) {
        const uint32_t byte = vat[i][size_t(tid / 2) * P];
        acc += fmaf(ps[i], float((byte >> (4 * (tid & 1))) & 15u), pl[i]);
      }
    m = mnew;
  }
  static_cast<T*>(p.out)[size_t(blockIdx.x) * D + tid] = from_f32<T>(m == -INFINITY ? 0.f : acc / l);
  if (tid == 0 && p.lse != nullptr) p.lse[blockIdx.x] = m == -INFINITY ? -INFINITY : m + logf(l);
}

// One warp per (sequence, KV head, token).
template <class T, int D>
__global__ void __launch_bounds__(256) weigh_kv4_rows_kernel(Kv4AttendParams p, uint32_t P) {
  __shared__ float qs[8][D];
  grid_dependency_wait();
  const uint32_t lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const uint32_t b = blockIdx.z, h = blockIdx.y;
  const uint32_t t = blockIdx.x * 8 + w;
  const uint32_t len = kv4_len(p.seq_lens, b, p.max_tokens);
  if (t == 0 && lane == 0 && __ldg(p.seq_lens + b) > p.max_tokens) atomicMax(&g_kvb_status, kKv4LenClamped);
  if (t >= len) return;
  const uint32_t page = p.table[size_t(b) * p.table_stride + t / P], s = t % P;
  if (page >= p.pool.pages) {
    if (lane == 0) atomicMax(&g_kvb_status, kKv4BadPage);
    return;
  }
  const uint64_t unit = uint64_t(page) * p.pool.kv_heads + h;
  const int32_t pk = p.pool.pos != nullptr ? p.pool.pos[unit * P + s] : int32_t(t);
  const uint32_t prefix = p.rule.prefix != nullptr ? p.rule.prefix[b] : 0u;
  float total = 0.f;
  for (uint32_t r = 0; r < p.rows; ++r)
    for (uint32_t g = 0; g < p.group; ++g) {
      const uint32_t head = h * p.group + g;
      for (int i = lane; i < D; i += 32)
        qs[w][i] = to_f32(static_cast<const T*>(p.q)[int64_t(b) * p.batch_stride + int64_t(r) * p.row_stride + head * D + i]);
      __syncwarp();
      if (lane == 0) {
        const int32_t pq = kv4_query_position(p.rule, b, r, p.rows, len);
        const float slope = p.rule.slopes != nullptr ? p.rule.slopes[head] : 0.f;
        const float x = kv4_score<D>(p, qs[w], P, unit, s, pk, pq, slope, prefix);
        if (x != -INFINITY) total += expf(x - p.lse_in[(size_t(b) * p.rows + r) * p.q_heads + head]);
      }
      __syncwarp();
    }
  if (lane == 0) p.weights[(int64_t(b) * p.pool.kv_heads + h) * p.weight_stride + t] += total;
}

}  // namespace kvb
