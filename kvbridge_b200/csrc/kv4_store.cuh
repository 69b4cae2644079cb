#pragma once
// Append to and read back from the 4-bit pool.
#include "kv4_common.cuh"

namespace kvb {

struct Kv4RowsParams {
  Kv4View pool;
  void* k;
  void* v;
  int64_t k_stride, v_stride;
  const int64_t* slots;
  const int32_t* positions;
  uint32_t tokens;
  uint64_t slots_total;  // pages * page_tokens
};

constexpr int kKv4RowWarps = 8;

// One warp per (token, KV head, K or V) row: lane l holds dims 2 l + 64 i
// and the next one, i.e. whole bytes of the packed row.
template <class T, int D>
__global__ void __launch_bounds__(32 * kKv4RowWarps) append_kv4_rows_kernel(Kv4RowsParams p, uint32_t P) {
  grid_dependency_wait();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t row = uint64_t(blockIdx.x) * kKv4RowWarps + (threadIdx.x >> 5);
  const uint32_t H = p.pool.kv_heads;
  if (row >= uint64_t(p.tokens) * H * 2) return;
  const bool is_v = row & 1;
  const uint64_t th = row >> 1;
  const uint32_t t = uint32_t(th / H), h = uint32_t(th % H);
  const int64_t slot = p.slots[t];
  if (slot < 0) return;
  if (uint64_t(slot) >= p.slots_total) {
    if (lane == 0) atomicMax(&g_kvb_status, kKv4BadSlot);
    return;
  }
  const T* x = static_cast<const T*>(is_v ? p.v : p.k) + int64_t(t) * (is_v ? p.v_stride : p.k_stride) +
               size_t(h) * D;
  float val[D / 32];
  float lo = INFINITY, hi = -INFINITY;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    val[i] = to_f32(x[64 * (i / 2) + 2 * lane + (i & 1)]);
    finite = finite && fabsf(val[i]) <= 3.402823466e38f;
    lo = fminf(lo, val[i]);
    hi = fmaxf(hi, val[i]);
  }
  lo = -warp_max(-lo);
  hi = warp_max(hi);
  const float scale = (hi - lo) * (1.0f / 15.0f);
  const bool ok = __all_sync(0xffffffffu, finite) && scale <= 3.402823466e38f;
  const float div = scale > 0.f ? scale : 1.0f;
  const uint64_t unit = uint64_t(slot) / P * H + h;
  const uint32_t s = uint32_t(uint64_t(slot) % P);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    uint32_t code[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      code[e] = ok ? uint32_t(fminf(fmaxf(rintf((val[2 * i + e] - lo) / div), 0.f), 15.f)) : 0u;
    const uint32_t pair = 32 * i + lane;  // d / 2
    uint8_t* dst = is_v ? p.pool.v + (unit * (D / 2) + pair) * P + s
                        : p.pool.k + (unit * P + s) * (D / 2) + pair;
    *dst = static_cast<uint8_t>(code[0] | (code[1] << 4));
  }
  if (lane == 0) {
    const float nan = __int_as_float(0x7fffffff);
    (is_v ? p.pool.vp : p.pool.kp)[unit * P + s] = ok ? make_float2(scale, lo) : make_float2(nan, nan);
    if (!is_v && p.pool.pos != nullptr) p.pool.pos[unit * P + s] = p.positions[t];
  }
}

template <class T, int D>
__global__ void __launch_bounds__(32 * kKv4RowWarps) load_kv4_rows_kernel(Kv4RowsParams p, uint32_t P) {
  grid_dependency_wait();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t row = uint64_t(blockIdx.x) * kKv4RowWarps + (threadIdx.x >> 5);
  const uint32_t H = p.pool.kv_heads;
  if (row >= uint64_t(p.tokens) * H * 2) return;
  const bool is_v = row & 1;
  const uint64_t th = row >> 1;
  const uint32_t t = uint32_t(th / H), h = uint32_t(th % H);
  const int64_t slot = p.slots[t];
  const bool ok = slot >= 0 && uint64_t(slot) < p.slots_total;
  if (slot >= 0 && !ok && lane == 0) atomicMax(&g_kvb_status, kKv4BadSlot);
  T* x = static_cast<T*>(is_v ? p.v : p.k) + int64_t(t) * (is_v ? p.v_stride : p.k_stride) + size_t(h) * D;
  const uint64_t unit = ok ? uint64_t(slot) / P * H + h : 0;
  const uint32_t s = ok ? uint32_t(uint64_t(slot) % P) : 0;
  const float2 par = ok ? (is_v ? p.pool.vp : p.pool.kp)[unit * P + s] : make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    const uint32_t pair = 32 * i + lane;
    const uint8_t* src = is_v ? p.pool.v + (unit * (D / 2) + pair) * P + s
                              : p.pool.k + (unit * P + s) * (D / 2) + pair;
    const uint32_t b = ok ? *src : 0u;
    x[2 * pair] = from_f32<T>(fmaf(par.x, float(b & 15u), par.y));
    x[2 * pair + 1] = from_f32<T>(fmaf(par.x, float(b >> 4), par.y));
  }
}

}  // namespace kvb
