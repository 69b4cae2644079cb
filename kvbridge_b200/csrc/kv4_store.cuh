#pragma once
// Append to and read back from the 4-bit pool (formats:
// include/kvbridge/attention_kv4.h): dense rows in, packed rows out, or the
// reverse. 65,536 bf16 tokens of 8 heads of 128 (344 MB) are appended in 114
// us, 3.0 TB/s, and loaded in 70 us, 4.9 TB/s (fp32, 612 MB: 111 and 125 us).
// The append of 16-bit rows is bound by instructions (two thirds of the issue
// slots, the conversions and the corrected quotients), fp32 rows and the load
// by HBM and its latency. Slots in no order take 318 and 165 us: V bytes of a
// token then lie in sectors of their own.
//
// One CTA of 8 warps per (KV head, tile of consecutive list tokens). A row
// (K or V of one token) is held by 8 or 16 lanes in runs of eight values = one
// packed word: one 16-byte load or store of 16-bit values, and a K row is
// stored by neighbouring lanes. Two runs a lane at dims 128 and 256, so that
// the row's reductions are shared by 16 values a lane. V is stored dim pair by dim pair, tokens side
// by side, so the tile's packed V words go through shared memory: where four
// list tokens in a row lie in four slots in a row from a multiple of four
// (any prompt but its ends), 4 x 4 byte transposes make whole words of four
// tokens; other tokens' bytes are moved one by one from where they are.
#include "kv4_common.cuh"

namespace kvb {

struct Kv4RowsParams {
  Kv4View pool;
  void* k;
  void* v;
  int64_t k_stride, v_stride;
  const int64_t* slots;
  const int32_t* positions;
  uint32_t tokens, page_tokens, log2_page;
  uint64_t slots_total;  // pages * page_tokens
  bool vector;           // 16-byte aligned rows
};

constexpr int kKv4StoreWarps = 8;

template <int D, int TILE>
struct Kv4Tile {
  // Element (unit * page_tokens + slot) of the params and positions, and the
  // byte of dim pair 0 in V; kNowhere: not in the pool.
  uint64_t at[TILE], v_at[TILE];
  uint32_t v[TILE][D / 8 + 1];  // packed V rows; the odd pitch spreads a column over the banks
  uint32_t slot[TILE];
  uint8_t quads[TILE / 4 + 1];  // first tokens of whole slot quads
  uint32_t count;               // of those
  uint32_t in_quad[(TILE + 31) / 32];  // tokens whose V is moved with its quad
};
constexpr uint64_t kNowhere = ~uint64_t(0);

// Where the tile's tokens of this CTA's head go, and its slot quads. Ends with
// a CTA barrier.
template <int D, int TILE>
__device__ __forceinline__ void kv4_map_tile(const Kv4RowsParams& p, uint32_t first, uint32_t h, Kv4Tile<D, TILE>& t) {
  const uint32_t P = p.page_tokens;
  for (uint32_t i = threadIdx.x; i < TILE; i += blockDim.x) {
    const int64_t slot = first + i < p.tokens ? kv4_load(p.slots + first + i) : -1;
    const bool ok = slot >= 0 && uint64_t(slot) < p.slots_total;
    if (slot >= 0 && !ok) atomicMax(&g_kvb_status, kKv4BadSlot);
    const uint32_t s = uint32_t(slot) & (P - 1);
    const uint64_t unit = (uint64_t(slot) >> p.log2_page) * p.pool.kv_heads + h;
    t.at[i] = ok ? unit * P + s : kNowhere;
    t.v_at[i] = unit * (D / 2) * P + s;
    t.slot[i] = s;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    uint32_t count = 0, before = 0;  // before: the quads of the 32 tokens before
#pragma unroll
    for (uint32_t base = 0; base < TILE; base += 32) {
      const uint32_t i = base + threadIdx.x;
      bool quad = i + 3 < TILE && t.at[i] != kNowhere && (t.slot[i] & 3) == 0;
      if (quad)  // neighbours of one page: a slot's element is the one before plus 1
        for (uint32_t k = 1; k < 4; ++k) quad = quad && t.at[i + k] == t.at[i] + k;
      const uint32_t mask = __ballot_sync(0xffffffffu, quad);
      if (quad) t.quads[count + __popc(mask & ((1u << threadIdx.x) - 1u))] = uint8_t(i);
      const uint64_t both = uint64_t(mask) << 32 | before;
      if (threadIdx.x == 0) t.in_quad[base / 32] = uint32_t((both | both << 1 | both << 2 | both << 3) >> 32);
      count += __popc(mask);
      before = mask;
    }
    if (threadIdx.x == 0) t.count = count;
  }
  __syncthreads();
}

// 4 x 4 bytes: byte j of w[i] becomes byte i of the result's word j.
__device__ __forceinline__ void transpose4(const uint32_t (&w)[4], uint32_t (&x)[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
  const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
  x[0] = __byte_perm(a, b, 0x5410), x[1] = __byte_perm(a, b, 0x7632);
  x[2] = __byte_perm(c, d, 0x5410), x[3] = __byte_perm(c, d, 0x7632);
}

// Eight values as they lie in memory.
template <class T>
struct alignas(16) Eight {
  T x[8];
};

template <class T>
__device__ __forceinline__ Eight<T> load_eight(const T* src, bool vector) {
  Eight<T> e;
  if (vector) {
    const uint4* s = reinterpret_cast<const uint4*>(src);
    uint4* d = reinterpret_cast<uint4*>(&e);
#pragma unroll
    for (int i = 0; i < int(sizeof(e) / 16); ++i) d[i] = kv4_stream(s + i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e.x[i] = src[i];
  }
  return e;
}

template <class T>
__device__ __forceinline__ void store_eight(T* dst, const Eight<T>& e, bool vector) {
  if (vector) {
    const uint4* s = reinterpret_cast<const uint4*>(&e);
#pragma unroll
    for (int i = 0; i < int(sizeof(e) / 16); ++i) __stcs(reinterpret_cast<uint4*>(dst) + i, s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = e.x[i];
  }
}

// The codes of eight values of a row, packed: rint of the correctly rounded
// quotient (x - lo) / scale, by Markstein's theorem: with y the correctly
// rounded 1 / b and q a faithful a / b, fma(fma(-q, b, a), y, q) is the
// correctly rounded quotient; a * y corrected once is faithful. (With a
// division each, or the product with a division near ties, which 16-bit values
// meet in four of five warps, the append of 65,536 tokens took 170 to 200 us
// where it took 144 with this.) Below
// 1e-30 the remainder may not be exact: divided.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], float lo, float scale) {
  uint32_t word = 0;
  const float div = scale > 0.f ? scale : 1.0f;
  if (div > 1e-30f) {
    const float y = 1.0f / div;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = x[e] - lo;
      float q = a * y;
      q = fmaf(fmaf(-q, div, a), y, q);
      q = fmaf(fmaf(-q, div, a), y, q);
      // at most 15; 1.5 * 2^23 leaves the integer in the low bits
      word = __funnelshift_r(word, __float_as_uint(q + 12582912.0f), 4);
    }
    return word;
  }
#pragma unroll 1
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float c = fminf(fmaxf(rintf(((half ? x[4 + e] : x[e]) - lo) / div), 0.f), 15.f);
      word = __funnelshift_r(word, uint32_t(c), 4);
    }
  return word;
}

// min and max that keep a NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// How a warp holds the V and then the K rows of its tokens: kRuns runs of
// eight values a lane, run r of lane `part` being run part + r * kLanes of the
// row; kBatch passes' loads are in flight together (MOST runs of a lane).
template <int D, int TILE, int MOST>
struct Kv4RowMap {
  static constexpr int kRuns = D == 64 ? 1 : 2, kLanes = D / 8 / kRuns, kRows = 32 / kLanes;
  static constexpr int kWarpTokens = TILE / kKv4StoreWarps, kPasses = 2 * kWarpTokens / kRows;
  static constexpr int kMost = MOST / kRuns;
  static constexpr int kBatch = kPasses < kMost ? kPasses : kMost;
  // Row of this lane in a pass: its token in the tile, and whether it is V.
  __device__ static uint32_t token(uint32_t pass, bool& is_v) {
    const uint32_t row = pass * kRows + (threadIdx.x & 31) / kLanes;
    is_v = row < kWarpTokens;
    return (threadIdx.x >> 5) * kWarpTokens + row % kWarpTokens;
  }
};

// Four CTAs an SM (64 registers a thread) hide the loads' latency: dim 256
// 235 us so, 256 us with what the compiler takes by itself.
template <class T, int D, int TILE>
__global__ void __launch_bounds__(32 * kKv4StoreWarps, 4) append_kv4_kernel(const Kv4RowsParams p) {
  using M = Kv4RowMap<D, TILE, 4>;
  __shared__ Kv4Tile<D, TILE> tile;
  const uint32_t part = threadIdx.x % M::kLanes;
  const uint32_t first = blockIdx.x * TILE, h = blockIdx.y, P = p.page_tokens;
  grid_launch_dependents();
  grid_dependency_wait();
  Eight<T> raw[M::kBatch][M::kRuns];
  auto load = [&](int pass) {
#pragma unroll
    for (int i = 0; i < M::kBatch; ++i) {
      bool is_v;
      const uint32_t t = M::token(pass + i, is_v);
      // (past the end: the last token again)
      const int64_t at = min(first + t, p.tokens - 1);
      const T* src = is_v ? static_cast<const T*>(p.v) + at * p.v_stride : static_cast<const T*>(p.k) + at * p.k_stride;
#pragma unroll
      for (int r = 0; r < M::kRuns; ++r)
        raw[i][r] = load_eight(src + size_t(h) * D + 8 * (part + r * M::kLanes), p.vector);
    }
  };
  load(0);
  kv4_map_tile(p, first, h, tile);
#pragma unroll 1
  for (int pass = 0; pass < M::kPasses; pass += M::kBatch) {
    if (pass != 0) load(pass);
#pragma unroll
    for (int i = 0; i < M::kBatch; ++i) {
      bool is_v;
      const uint32_t t = M::token(pass + i, is_v);
      float x[M::kRuns][8];
#pragma unroll
      for (int r = 0; r < M::kRuns; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[r][e] = to_f32(raw[i][r].x[e]);
      float lo = x[0][0], hi = x[0][0];
#pragma unroll
      for (int r = 0; r < M::kRuns; ++r)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          lo = min_nan(lo, x[r][e]);
          hi = max_nan(hi, x[r][e]);
        }
#pragma unroll
      for (int o = 1; o < M::kLanes; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      // NaN for a NaN in the row and for equal infinities, infinite for others
      float scale = (hi - lo) * (1.0f / 15.0f);
      const bool ok = scale <= 3.402823466e38f;
      if (!ok) scale = lo = __int_as_float(0x7fffffff);
      const uint64_t at = tile.at[t];
      if (at == kNowhere) continue;
      const bool in_quad = tile.in_quad[t / 32] >> (t % 32) & 1u;
#pragma unroll
      for (int r = 0; r < M::kRuns; ++r) {
        const uint32_t word = ok ? kv4_codes(x[r], lo, scale) : 0u, q = part + r * M::kLanes;
        if (!is_v) {
          reinterpret_cast<uint32_t*>(p.pool.k)[at * (D / 8) + q] = word;
        } else if (in_quad) {
          tile.v[t][q] = word;
        } else {
          uint8_t* dst = p.pool.v + tile.v_at[t] + 4 * q * P;
#pragma unroll
          for (int j = 0; j < 4; ++j) dst[j * P] = uint8_t(word >> (8 * j));
        }
      }
      if (part == 0) {
        (is_v ? p.pool.vp : p.pool.kp)[at] = make_float2(scale, lo);
        if (!is_v && p.pool.pos != nullptr) p.pool.pos[at] = kv4_load(p.positions + first + t);
      }
    }
  }
  const uint32_t quads = tile.count;
  if (quads == 0) return;
  __syncthreads();
  // V: neighbouring threads take neighbouring quads of four dim pairs.
  for (uint32_t i = threadIdx.x; i < TILE / 4 * (D / 8); i += 32 * kKv4StoreWarps) {
    if (i % (TILE / 4) >= quads) continue;
    const uint32_t t = tile.quads[i % (TILE / 4)], q = i / (TILE / 4);
    const uint32_t w[4] = {tile.v[t][q], tile.v[t + 1][q], tile.v[t + 2][q], tile.v[t + 3][q]};
    uint32_t x[4];
    transpose4(w, x);
    uint8_t* dst = p.pool.v + tile.v_at[t] + 4 * q * P;
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(dst + j * P) = x[j];
  }
}

// The inverse. V words are fetched before the K rows are written and turned
// after, so that both halves' reads are in flight together.
template <class T, int D, int TILE>
__global__ void __launch_bounds__(32 * kKv4StoreWarps) load_kv4_kernel(const Kv4RowsParams p) {
  using M = Kv4RowMap<D, TILE, sizeof(T) == 2 ? 8 : 4>;
  __shared__ Kv4Tile<D, TILE> tile;
  const uint32_t part = threadIdx.x % M::kLanes;
  const uint32_t first = blockIdx.x * TILE, h = blockIdx.y, P = p.page_tokens;
  grid_launch_dependents();
  grid_dependency_wait();
  kv4_map_tile(p, first, h, tile);
  // V quads: fetched now, transposed into shared memory once K is done.
  constexpr int kItems = (TILE / 4 * (D / 8) + 32 * kKv4StoreWarps - 1) / (32 * kKv4StoreWarps);
  const uint32_t quads = tile.count;
  uint32_t w[kItems][4];
#pragma unroll
  for (int n = 0; n < kItems; ++n) {
    const uint32_t i = threadIdx.x + n * 32 * kKv4StoreWarps, q = i / (TILE / 4);
    if (i % (TILE / 4) >= quads || q >= D / 8) continue;
    const uint8_t* src = p.pool.v + tile.v_at[tile.quads[i % (TILE / 4)]] + 4 * q * P;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[n][j] = kv4_stream(reinterpret_cast<const uint32_t*>(src + j * P));
  }
  constexpr int kFirstK = M::kWarpTokens / M::kRows;  // the pass with the first K rows
  constexpr int kHalf = kFirstK == 0 ? M::kPasses : kFirstK, kBatch = kHalf < M::kBatch ? kHalf : M::kBatch;
  auto rows = [&](int from, int to, bool want_v) {
#pragma unroll 1
    for (int pass = from; pass < to; pass += kBatch) {
      uint32_t word[kBatch][M::kRuns] = {};
      float2 par[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        bool is_v;
        const uint32_t t = M::token(pass + i, is_v);
        const uint64_t at = tile.at[t];
        par[i] = make_float2(0.f, 0.f);  // zeros where the slot is not in the pool
        if (is_v != want_v || at == kNowhere) continue;
        const bool in_quad = tile.in_quad[t / 32] >> (t % 32) & 1u;
        par[i] = kv4_load((is_v ? p.pool.vp : p.pool.kp) + at);
#pragma unroll
        for (int r = 0; r < M::kRuns; ++r) {
          const uint32_t q = part + r * M::kLanes;
          if (!is_v) {
            word[i][r] = kv4_stream(reinterpret_cast<const uint32_t*>(p.pool.k) + at * (D / 8) + q);
          } else if (in_quad) {
            word[i][r] = tile.v[t][q];
          } else {
            const uint8_t* src = p.pool.v + tile.v_at[t] + 4 * q * P;
#pragma unroll
            for (int j = 0; j < 4; ++j) word[i][r] |= uint32_t(src[j * P]) << (8 * j);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        bool is_v;
        const uint32_t t = M::token(pass + i, is_v);
        if (is_v != want_v || first + t >= p.tokens) continue;
        T* dst = is_v ? static_cast<T*>(p.v) + int64_t(first + t) * p.v_stride
                      : static_cast<T*>(p.k) + int64_t(first + t) * p.k_stride;
#pragma unroll
        for (int r = 0; r < M::kRuns; ++r) {
          const uint32_t even = word[i][r] & 0x0f0f0f0fu, odd = word[i][r] >> 4 & 0x0f0f0f0fu;
          Eight<T> out;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            // the code in the low byte of 2^23
            const float code = __uint_as_float(__byte_perm(e & 1 ? odd : even, 0x4B000000u, 0x7650 + e / 2)) - 8388608.0f;
            out.x[e] = from_f32<T>(fmaf(par[i].x, code, par[i].y));
          }
          store_eight(dst + size_t(h) * D + 8 * (part + r * M::kLanes), out, p.vector);
        }
      }
    }
  };
  rows(kFirstK, M::kPasses, false);
#pragma unroll
  for (int n = 0; n < kItems; ++n) {
    const uint32_t i = threadIdx.x + n * 32 * kKv4StoreWarps, q = i / (TILE / 4);
    if (i % (TILE / 4) >= quads || q >= D / 8) continue;
    const uint32_t t = tile.quads[i % (TILE / 4)];
    uint32_t x[4];
    transpose4(w[n], x);
#pragma unroll
    for (int j = 0; j < 4; ++j) tile.v[t + j][q] = x[j];
  }
  if (quads != 0) __syncthreads();
  rows(0, kHalf, true);
}

}  // namespace kvb
