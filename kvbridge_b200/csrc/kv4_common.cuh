#pragma once
// Device view of the 4-bit pool and the score rule shared by the kv4 kernels
// (formats: include/kvbridge/attention_kv4.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kvb_device.cuh"

namespace kvb {

// Codes in the device status word beside those of the other kernels.
enum : int {
  kKv4BadPage = 4,
  kKv4LenClamped = 5,
  kKv4BadSlot = 6,
  kKv4BadKept = 8,
};

// Loads of what the preceding kernel may have written. These kernels start
// before it has ended (programmatic dependent launch), so nothing of theirs is
// read-only for their lifetime, as the non-coherent load instructions ask.
template <class T>
__device__ __forceinline__ T kv4_load(const T* p) {
  return *p;
}
// The same for data used once.
template <class T>
__device__ __forceinline__ T kv4_stream(const T* p) {
  return __ldcs(p);
}

struct Kv4View {
  uint8_t* k;
  uint8_t* v;
  float2* kp;  // {scale, lo}
  float2* vp;
  int32_t* pos;  // or null
  uint32_t kv_heads, pages;
};

struct Kv4Rule {
  float scale, softcap;
  uint32_t window;
  const float* slopes;
  const uint32_t* prefix;
  const int32_t* q_pos;
};

// Row r of `rows` query rows of a sequence of `len` tokens.
__device__ __forceinline__ int32_t kv4_query_position(const Kv4Rule& rule, uint32_t b, uint32_t r,
                                                      uint32_t rows, uint32_t len) {
  return rule.q_pos != nullptr ? kv4_load(rule.q_pos + size_t(b) * rows + r)
                               : int32_t(len) - int32_t(rows) + int32_t(r);
}

// Positions of tokens are not negative; a query row's may be (more rows than
// tokens), and pq - pk is only formed where pk <= pq. A prefix of 2^31 or more
// is a negative int32, below which nothing lies.
__device__ __forceinline__ bool kv4_visible(int32_t pk, int32_t pq, uint32_t window,
                                            int32_t prefix) {
  const bool past = pk <= pq && (window == 0 || uint32_t(pq - pk) < window);
  return past || pk < prefix;
}

__device__ __forceinline__ uint32_t kv4_len(const uint32_t* seq_lens, uint32_t b,
                                            uint32_t max_tokens) {
  const uint32_t len = kv4_load(seq_lens + b);
  return len > max_tokens ? max_tokens : len;
}

template <class T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else return static_cast<float>(x);
}
template <class T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

// 16 bytes global -> shared, asynchronously and past L1.
__device__ __forceinline__ void copy16_async(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the latest `N` committed groups of this thread have landed.
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

}  // namespace kvb
