// Launchers of the 4-bit cache operators (include/kvbridge/attention_kv4.h).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <limits>
#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <utility>
#include <type_traits>

#include "kvbridge/attention_b200.h"
#include "kvbridge/attention_kv4.h"
#include "kv4_attend.cuh"
#include "kv4_evict.cuh"
#include "kv4_store.cuh"
#include "launch_checks.h"
#include "launch_internal.h"

namespace kvbridge {
namespace {

using detail::aligned_to;
using detail::cuda_ok;

// Whether this process has launched a kernel of this module (or captured one):
// until then reading the status leaves the module unloaded.
std::atomic<bool> g_launched{false};

void launch_kernel_pdl(const void* fn, dim3 grid, dim3 block, uint32_t smem, cudaStream_t stream, void** args,
                       const char* what) {
  g_launched.store(true, std::memory_order_relaxed);
  detail::launch_kernel_pdl(fn, grid, block, smem, stream, args, what);
}

constexpr uint32_t kMaxColumns = 128;  // query rows x heads of a KV head

void require(const char* error) {
  if (error != nullptr) throw std::invalid_argument(error);
}

uintptr_t type_bytes(Kv4Type t) { return t == Kv4Type::f32 ? 4 : 2; }

bool type_ok(Kv4Type t) { return t == Kv4Type::f32 || t == Kv4Type::f16 || t == Kv4Type::bf16; }

void check_pool(const Kv4Pool& p) {
  require(kv4_pool_error(p));
  if (!p.k || !p.v || !p.k_params || !p.v_params)
    throw std::invalid_argument("kv4 pool buffers must be non-null");
  if (!aligned_to(p.k, 16) || !aligned_to(p.v, 16) || !aligned_to(p.k_params, 16) ||
      !aligned_to(p.v_params, 16) || !aligned_to(p.positions, 16))
    throw std::invalid_argument("kv4 pool buffers must be 16-byte aligned");
}

kvb::Kv4View view(const Kv4Pool& p) {
  return kvb::Kv4View{p.k, p.v, reinterpret_cast<float2*>(p.k_params),
                      reinterpret_cast<float2*>(p.v_params), p.positions, p.kv_heads, p.pages};
}

uint32_t log2_page(const Kv4Pool& p) { return p.page_tokens == 64 ? 6 : p.page_tokens == 32 ? 5 : 4; }

// Calls f(integral_constant<int, D>) with the pool's head dim.
template <class F>
auto by_dim(uint32_t dim, F&& f) {
  if (dim == 64) return f(std::integral_constant<int, 64>{});
  if (dim == 128) return f(std::integral_constant<int, 128>{});
  return f(std::integral_constant<int, 256>{});
}

// Calls f(T{}) with the C++ type of a Kv4Type.
template <class F>
auto by_type(Kv4Type type, F&& f) {
  if (type == Kv4Type::f32) return f(float{});
  if (type == Kv4Type::f16) return f(__half{});
  return f(__nv_bfloat16{});
}

}  // namespace

const char* kv4_pool_error(const Kv4Pool& p) noexcept {
  if (p.kv_heads == 0 || p.kv_heads > 65535) return "kv_heads must be in [1, 65535]";
  if (p.dim != 64 && p.dim != 128 && p.dim != 256) return "kv4 needs dim 64, 128 or 256";
  if (p.page_tokens != 16 && p.page_tokens != 32 && p.page_tokens != 64)
    return "kv4 needs page_tokens 16, 32 or 64";
  if (p.pages == 0) return "pages must be positive";
  if (uint64_t(p.pages) * p.kv_heads >= 0xffffffffull) return "kv4 pool extent too large: pages * kv_heads";
  return nullptr;
}

namespace {

// Shared checks of append_kv4 and load_kv4; false if there is nothing to do.
bool check_rows(const Kv4Pool& pool, const Kv4Rows& rows) {
  require(kv4_pool_error(pool));
  if (!type_ok(rows.type)) throw std::invalid_argument("unknown element type");
  if (rows.tokens == 0) return false;
  check_pool(pool);
  if (!rows.k || !rows.v || !rows.slots)
    throw std::invalid_argument("kv4 rows and slots must be non-null device buffers");
  const uintptr_t bytes = type_bytes(rows.type);
  if (!aligned_to(rows.k, bytes) || !aligned_to(rows.v, bytes) || !aligned_to(rows.slots, 8) ||
      !aligned_to(rows.positions, 4))
    throw std::invalid_argument("kv4 rows, slots and positions must be aligned to their elements");
  const int64_t width = int64_t(pool.kv_heads) * pool.dim;
  if (rows.tokens > 1 && (rows.k_stride < width || rows.v_stride < width))
    throw std::invalid_argument("kv4 row strides must be at least kv_heads * dim");
  return true;
}

kvb::Kv4RowsParams rows_params(const Kv4Pool& pool, const Kv4Rows& rows) {
  const int64_t per = int64_t(16 / type_bytes(rows.type));  // elements of a vector access
  const bool vector = aligned_to(rows.k, 16) && aligned_to(rows.v, 16) && rows.k_stride % per == 0 &&
                      rows.v_stride % per == 0;
  return kvb::Kv4RowsParams{view(pool),
                            rows.k,
                            rows.v,
                            rows.k_stride,
                            rows.v_stride,
                            rows.slots,
                            rows.positions,
                            rows.tokens,
                            pool.page_tokens,
                            log2_page(pool),
                            uint64_t(pool.pages) * pool.page_tokens,
                            vector};
}

// Tokens a CTA: 16 where 64 would give an SM less than two CTAs (64 tokens
// appended and loaded 6.9 us for 10.3, 1,024 tokens 18 us for 32); else 64, but
// 32 to append rows of dim 128, whose loads are then one batch a lane (65,536
// bf16 tokens on 8 heads 114 us for 129; fp32 111 for 113; dims 64 and 256 the
// other way round, 70 us for 85 and 235 for 294; to load, 64 is better at any
// dim, at 128 69 us for 85).
bool small_tiles(const Kv4Pool& pool, const Kv4Rows& rows) {
  return uint64_t((rows.tokens + 63) / 64) * pool.kv_heads < uint64_t(2 * detail::device_sms());
}

constexpr uint32_t append_tile(uint32_t dim) { return dim == 128 ? 32 : 64; }

template <class Kernel>
void launch_rows(const Kv4Pool& pool, const Kv4Rows& rows, uint32_t large, cudaStream_t stream, const char* what,
                 Kernel&& kernel) {
  kvb::Kv4RowsParams prm = rows_params(pool, rows);
  const bool small = small_tiles(pool, rows);
  const uint32_t tile = small ? 16 : large;
  const void* fn = by_dim(pool.dim, [&](auto d) { return by_type(rows.type, [&](auto t) { return kernel(d, t, small); }); });
  void* args[] = {&prm};
  launch_kernel_pdl(fn, dim3((rows.tokens + tile - 1) / tile, pool.kv_heads), dim3(32 * kvb::kKv4StoreWarps), 0, stream,
                    args, what);
}

}  // namespace

void append_kv4(const Kv4Pool& pool, const Kv4Rows& rows, cudaStream_t stream) {
  if (!check_rows(pool, rows)) return;
  if (pool.positions != nullptr && rows.positions == nullptr)
    throw std::invalid_argument("the pool keeps positions: append_kv4 needs the rows' positions");
  launch_rows(pool, rows, append_tile(pool.dim), stream, "kv4 append launch", [](auto d, auto t, bool small) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return small ? reinterpret_cast<const void*>(&kvb::append_kv4_kernel<T, D, 16>)
                 : reinterpret_cast<const void*>(&kvb::append_kv4_kernel<T, D, append_tile(D)>);
  });
}

void load_kv4(const Kv4Pool& pool, const Kv4Rows& rows, cudaStream_t stream) {
  if (!check_rows(pool, rows)) return;
  launch_rows(pool, rows, 64, stream, "kv4 load launch", [](auto d, auto t, bool small) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return small ? reinterpret_cast<const void*>(&kvb::load_kv4_kernel<T, D, 16>)
                 : reinterpret_cast<const void*>(&kvb::load_kv4_kernel<T, D, 64>);
  });
}

// ---------------------------------------------------------------------------
// Attention and weights.

const char* kv4_query_error(const Kv4Pool& pool, const Kv4Query& q) noexcept {
  if (const char* e = kv4_pool_error(pool)) return e;
  if (q.batch == 0 || q.rows == 0 || q.q_heads == 0) return "batch, rows and q_heads must be positive";
  if (q.q_heads % pool.kv_heads) return "q_heads must be divisible by kv_heads";
  if (uint64_t(q.rows) * (q.q_heads / pool.kv_heads) > kMaxColumns)
    return "rows * (q_heads / kv_heads) must be at most 128";
  if (!type_ok(q.type)) return "unknown element type";
  if (q.batch > 65535) return "batch must be at most 65535";
  if (q.table_stride == 0) return "table_stride must be positive";
  if (q.max_tokens > 0x7fffffffu - 65536u) return "max_tokens must be below 2^31 - 65536";
  if (!std::isfinite(q.scale)) return "score scale must be finite";
  if (!std::isfinite(q.softcap) || q.softcap < 0.f) return "softcap must be finite and not negative";
  if (uint64_t(q.batch) * q.rows * q.q_heads > 0x7fffffffull) return "batch/row/head product too large";
  if (q.batch_stride < 0 || q.row_stride < 0) return "query strides must not be negative";
  return nullptr;
}

namespace {

kvb::Kv4AttendParams check_query(const Kv4Pool& pool, const Kv4Query& q) {
  require(kv4_query_error(pool, q));
  check_pool(pool);
  if (!q.q || !q.seq_lens || !q.block_table)
    throw std::invalid_argument("kv4 query, seq_lens and block_table must be non-null");
  if (!aligned_to(q.q, type_bytes(q.type)) || !aligned_to(q.seq_lens, 4) ||
      !aligned_to(q.block_table, 4) || !aligned_to(q.q_positions, 4) || !aligned_to(q.slopes, 4) ||
      !aligned_to(q.prefix_lens, 4))
    throw std::invalid_argument("kv4 query buffers must be aligned to their elements");
  if (pool.positions != nullptr && q.q_positions == nullptr)
    throw std::invalid_argument("the pool keeps positions: the query needs q_positions");
  kvb::Kv4AttendParams prm{};
  prm.pool = view(pool);
  prm.rule = kvb::Kv4Rule{q.scale, q.softcap, q.window, q.slopes, q.prefix_lens, q.q_positions};
  prm.q = q.q;
  prm.batch_stride = q.batch_stride;
  prm.row_stride = q.row_stride;
  prm.seq_lens = q.seq_lens;
  prm.table = q.block_table;
  prm.batch = q.batch;
  prm.rows = q.rows;
  prm.q_heads = q.q_heads;
  prm.group = q.q_heads / pool.kv_heads;
  prm.table_stride = q.table_stride;
  prm.page_tokens = pool.page_tokens;
  prm.log2_page = log2_page(pool);
  prm.type = int32_t(q.type);
  const int64_t per = int64_t(16 / type_bytes(q.type));  // elements of a vector load
  prm.vector_q = aligned_to(q.q, 16) && q.batch_stride % per == 0 && q.row_stride % per == 0;
  prm.max_tokens = uint32_t(std::min<uint64_t>(q.max_tokens, uint64_t(q.table_stride) * pool.page_tokens));
  return prm;
}

}  // namespace

namespace {

// One attention or weights kernel: its entry point and its shared memory.
struct Kv4Kernel {
  const void* fn;
  uint32_t smem;
};

// CTAs of 128 threads an SM, i.e. the register cap: 128 registers at four,
// 168 at three, 255 at two. (Dim 128, 8 columns: three CTAs 83 us for 16x16K
// tokens, four 94 us with 160 bytes of spills; 4 columns: 1x64K 26.6 us at
// three, 28.0 us at four. Weights of 32 sequences of 1K to 32K tokens, 8
// columns: three (48 to 80 bytes of spills) 82 us, with cap and bias 115 us; four
// (64 to 128 bytes) 81 and 117 us; 1x64K, 4 columns, which spill at four alone,
// 13.1 against 13.4 us.)
constexpr int attend_ctas(int dim) { return dim == 256 ? 2 : dim == 64 ? 4 : 3; }

template <int D, int C, int PD, int RULES>
Kv4Kernel attend_kernel() {
  return {reinterpret_cast<const void*>(&kvb::attend_kv4_kernel<D, C, PD, attend_ctas(D), RULES>),
          kvb::Kv4Smem<D, true>::kBytes};
}

template <int D, int C, int RULES>
Kv4Kernel weigh_kernel() {
  return {reinterpret_cast<const void*>(&kvb::weigh_kv4_kernel<D, C, attend_ctas(D), RULES>),
          kvb::Kv4Smem<D, false>::kBytes};
}

int rules_of(const Kv4Pool& pool, const Kv4Query& q) {
  if (q.softcap > 0.f || q.slopes || q.q_positions || pool.positions) return kvb::kRulesAll;
  return q.window != 0 || q.prefix_lens ? kvb::kRulesMask : kvb::kRulesNone;
}

// Calls f(integral_constant<int, RULES>).
template <class F>
auto by_rules(int rules, F&& f) {
  if (rules == kvb::kRulesNone) return f(std::integral_constant<int, kvb::kRulesNone>{});
  if (rules == kvb::kRulesMask) return f(std::integral_constant<int, kvb::kRulesMask>{});
  return f(std::integral_constant<int, kvb::kRulesAll>{});
}

// Query columns a segment: 4 where all of a KV head's fit (32 sequences of 1K to
// 32K tokens, group 4: 106 us, with 8 half of whose rows are idle 126 us), else 8
// (64 x 16K tokens, group 8: 248 us, with 4 and every page read twice 454 us).
uint32_t segment_columns(const Kv4Pool& pool, const Kv4Query& q) {
  return q.rows * (q.q_heads / pool.kv_heads) <= 4 ? 4 : 8;
}

Kv4Kernel attend_kernel(uint32_t dim, uint32_t cols, bool f32, int rules) {
  return by_dim(dim, [&](auto d) {
    return by_rules(rules, [&](auto r) {
      constexpr int D = decltype(d)::value, RULES = decltype(r)::value;
      return cols == 4 ? f32 ? attend_kernel<D, 4, 3, RULES>() : attend_kernel<D, 4, 2, RULES>()
             : f32     ? attend_kernel<D, 8, 3, RULES>()
                       : attend_kernel<D, 8, 2, RULES>();
    });
  });
}

Kv4Kernel weigh_kernel(uint32_t dim, uint32_t cols, int rules) {
  return by_dim(dim, [&](auto d) {
    return by_rules(rules, [&](auto r) {
      constexpr int D = decltype(d)::value, RULES = decltype(r)::value;
      return cols == 4 ? weigh_kernel<D, 4, RULES>() : weigh_kernel<D, 8, RULES>();
    });
  });
}

// CTAs of a kernel that the current device holds at once. The first use on a
// device also raises the kernel's shared-memory limit.
uint32_t resident_ctas(const Kv4Kernel& k, int threads = kvb::kKv4Threads) {
  static std::mutex mu;
  static std::map<std::pair<int, const void*>, uint32_t> cache;
  int dev = 0;
  cuda_ok(cudaGetDevice(&dev), "cudaGetDevice");
  std::lock_guard<std::mutex> lock(mu);
  const auto key = std::make_pair(dev, k.fn);
  const auto it = cache.find(key);
  if (it != cache.end()) return it->second;
  cuda_ok(cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(k.smem)),
          "kv4 kernel shared-memory opt-in");
  cuda_ok(cudaFuncSetAttribute(k.fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                               int(cudaSharedmemCarveoutMaxShared)),
          "kv4 kernel carveout");
  int blocks = 0;
  cuda_ok(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, k.fn, threads, k.smem), "occupancy query");
  const uint32_t ctas = uint32_t(std::max(blocks, 1) * detail::device_sms());
  cache.emplace(key, ctas);
  return ctas;
}

// CTAs of a call whose segments have at most max_tokens tokens: a full wave,
// or fewer where there are fewer stages than warps.
uint32_t split_ctas(const Kv4Kernel& k, uint64_t segments, uint32_t max_tokens) {
  const uint64_t stages = segments * ((uint64_t(max_tokens) + kvb::kStageTokens - 1) / kvb::kStageTokens);
  const uint64_t most = (stages + kvb::kKv4Warps - 1) / kvb::kKv4Warps;
  return uint32_t(std::max<uint64_t>(1, std::min<uint64_t>(resident_ctas(k), most)));
}

struct AttendPlan {
  Kv4Kernel kernel;
  int rules;
  bool direct, many, most;
  uint32_t cols, col_groups, segments, ctas, workers;
  size_t ml_offset, warps_offset, bytes;  // of the workspace
};

// Short sequences: one warp per segment writes the result, nothing is merged.
// (64 sequences of 128 tokens 9.6 us, split and merged 11.4 us, and one launch
// less; eight of up to 256 tokens 12.3 us so and 9.0 us split.)
constexpr uint32_t kDirectTokens = 128;

AttendPlan plan_attention(const Kv4Pool& pool, const Kv4Query& q) {
  AttendPlan a{};
  a.rules = rules_of(pool, q);
  const bool f32 = q.type == Kv4Type::f32;
  const uint32_t cols = a.cols = segment_columns(pool, q), all = q.rows * (q.q_heads / pool.kv_heads);
  a.kernel = attend_kernel(pool.dim, cols, f32, a.rules);
  a.col_groups = (all + cols - 1) / cols;
  a.segments = q.batch * pool.kv_heads * a.col_groups;
  a.direct = q.max_tokens <= kDirectTokens;
  if (a.direct) {
    resident_ctas(a.kernel);
    a.workers = a.segments;
    a.ctas = (a.segments + kvb::kKv4Warps - 1) / kvb::kKv4Warps;
    a.bytes = 16;
    return a;
  }
  // At most 512 partials a segment: one KV head of 131,072 tokens takes 18.5 us
  // so, 26.9 us with a full wave's 1,776 partials to merge.
  const uint64_t capped = uint64_t(512 / kvb::kKv4Warps) * a.segments;
  a.ctas = uint32_t(std::min<uint64_t>(split_ctas(a.kernel, a.segments, q.max_tokens), capped));
  a.workers = a.ctas * kvb::kKv4Warps;
  // A warp reads 32 partials a round; from about 24 on a CTA a row is faster.
  a.many = a.workers > 24 * a.segments;
  // More than a round of eight a warp (1x64K tokens, 222 a row: 25.2 against 23.6 us).
  a.most = a.workers > (pool.dim == 256 ? 64 : 128) * a.segments;
  const size_t slots = size_t(a.workers) + a.segments;
  a.ml_offset = slots * cols * pool.dim * sizeof(float);
  a.warps_offset = a.ml_offset + slots * cols * sizeof(float2);
  a.bytes = a.warps_offset + size_t(a.segments) * sizeof(uint2);
  return a;
}

}  // namespace

size_t attention_kv4_workspace_bytes(const Kv4Pool& pool, const Kv4Query& q) {
  require(kv4_query_error(pool, q));
  return plan_attention(pool, q).bytes;
}

void launch_attention_kv4(const Kv4Pool& pool, const Kv4Query& q, void* workspace,
                          size_t workspace_bytes, void* out, float* lse, cudaStream_t stream) {
  kvb::Kv4AttendParams prm = check_query(pool, q);
  if (!workspace || !out) throw std::invalid_argument("kv4 workspace and output must be non-null");
  if (!aligned_to(workspace, 16) || !aligned_to(out, type_bytes(q.type)) || !aligned_to(lse, 4))
    throw std::invalid_argument("kv4 workspace must be 16-byte aligned, outputs to their elements");
  const AttendPlan a = plan_attention(pool, q);
  if (workspace_bytes < a.bytes)
    throw std::invalid_argument("workspace smaller than attention_kv4_workspace_bytes(pool, query)");
  prm.col_groups = a.col_groups;
  prm.workers = a.workers;
  prm.direct = a.direct;
  prm.part = static_cast<float*>(workspace);
  prm.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + a.ml_offset);
  prm.seg_warps = reinterpret_cast<uint2*>(static_cast<uint8_t*>(workspace) + a.warps_offset);
  prm.out = out;
  prm.lse = lse;
  void* args[] = {&prm};
  launch_kernel_pdl(a.kernel.fn, dim3(a.ctas), dim3(kvb::kKv4Threads), a.kernel.smem, stream, args,
                    "kv4 attention launch");
  if (a.direct) return;
  uint32_t cols = a.cols;
  void* merge_args[] = {&prm, &cols};
  const void* merge = by_dim(pool.dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    return by_rules(a.rules, [&](auto r) {
      constexpr int RULES = decltype(r)::value;
      return !a.many  ? reinterpret_cast<const void*>(&kvb::merge_kv4_kernel<D, RULES, false, 8>)
             : a.most ? reinterpret_cast<const void*>(&kvb::merge_kv4_kernel<D, RULES, true, 16>)
                      : reinterpret_cast<const void*>(&kvb::merge_kv4_kernel<D, RULES, true, 8>);
    });
  });
  const uint32_t rows = q.batch * q.rows * q.q_heads;
  launch_kernel_pdl(merge, dim3(a.many ? rows : (rows + kvb::kKv4MergeWarps - 1) / kvb::kKv4MergeWarps),
                    dim3(32 * kvb::kKv4MergeWarps), 0, stream, merge_args, "kv4 merge launch");
}

void accumulate_weights_kv4(const Kv4Pool& pool, const Kv4Query& q, const float* lse, float* weights,
                            int64_t weight_stride, cudaStream_t stream) {
  kvb::Kv4AttendParams prm = check_query(pool, q);
  if (!lse || !weights) throw std::invalid_argument("kv4 lse and weights must be non-null");
  if (!aligned_to(lse, 4) || !aligned_to(weights, 4))
    throw std::invalid_argument("kv4 lse and weights must be 4-byte aligned");
  if (weight_stride < int64_t(prm.max_tokens))
    throw std::invalid_argument("weight_stride must be at least max_tokens");
  if (prm.max_tokens == 0) return;
  const uint32_t cols = segment_columns(pool, q), groups = (q.rows * prm.group + cols - 1) / cols;
  const Kv4Kernel k = weigh_kernel(pool.dim, cols, rules_of(pool, q));
  prm.col_groups = 1;
  const uint32_t ctas = split_ctas(k, uint64_t(q.batch) * pool.kv_heads, prm.max_tokens);
  prm.workers = ctas * kvb::kKv4Warps;
  prm.lse_in = lse;
  prm.weights = weights;
  prm.weight_stride = weight_stride;
  for (uint32_t group = 0; group < groups; ++group) {
    void* args[] = {&prm, &group};
    launch_kernel_pdl(k.fn, dim3(ctas), dim3(kvb::kKv4Threads), k.smem, stream, args, "kv4 weights launch");
  }
}

// ---------------------------------------------------------------------------
// Eviction.

const char* kv4_eviction_error(const Kv4Eviction& e) noexcept {
  if (e.batch == 0 || e.batch > 65535) return "batch must be in [1, 65535]";
  if (e.kv_heads == 0 || e.kv_heads > 65535) return "kv_heads must be in [1, 65535]";
  if (uint64_t(e.batch) * e.kv_heads > 0x7fffffffull) return "batch/head product too large";
  if (e.max_tokens > 0x7fffffffu - 65536u) return "max_tokens must be below 2^31 - 65536";
  if (e.budget == 0 || e.budget > 0x7fffffffu - 65536u) return "budget must be positive and below 2^31 - 65536";
  if (uint64_t(e.sinks) + e.recent > e.budget) return "sinks + recent must not exceed budget";
  if (e.weight_stride < int64_t(e.max_tokens)) return "weight_stride must be at least max_tokens";
  return nullptr;
}

namespace {

void check_eviction(const Kv4Eviction& e) {
  require(kv4_eviction_error(e));
  if (!e.seq_lens || !e.weights) throw std::invalid_argument("eviction seq_lens and weights must be non-null");
  if (!aligned_to(e.seq_lens, 4) || !aligned_to(e.weights, 4))
    throw std::invalid_argument("eviction seq_lens and weights must be 4-byte aligned");
}

// Whether some of `rows` rows of `a` (a_width floats each, a_stride apart) share
// a float with some of `b`'s.
bool rows_overlap(const float* a, int64_t a_stride, int64_t a_width, const float* b, int64_t b_stride, int64_t b_width,
                  int64_t rows) {
  const int64_t from = (int64_t(reinterpret_cast<uintptr_t>(b)) - int64_t(reinterpret_cast<uintptr_t>(a))) / int64_t(sizeof(float));
  if (a_width == 0 || b_width == 0 || from >= (rows - 1) * a_stride + a_width || -from >= (rows - 1) * b_stride + b_width)
    return false;
  for (int64_t j = 0; j < rows; ++j) {
    const int64_t start = from + j * b_stride;  // from a's first float
    const int64_t i = start < a_width ? 0 : (start - a_width) / a_stride + 1;  // the first row of a that ends after it
    if (i < rows && i * a_stride < start + b_width) return true;
  }
  return false;
}

}  // namespace

void select_tokens(const Kv4Eviction& e, int32_t* keep, uint32_t* kept_lens, cudaStream_t stream) {
  check_eviction(e);
  if (!keep || !kept_lens) throw std::invalid_argument("keep and kept_lens must be non-null");
  if (!aligned_to(keep, 4) || !aligned_to(kept_lens, 4))
    throw std::invalid_argument("keep and kept_lens must be 4-byte aligned");
  // Every CTA of a sequence reads its length, one writes what is kept of it.
  if (kept_lens < e.seq_lens + e.batch && e.seq_lens < kept_lens + e.batch)
    throw std::invalid_argument("kept_lens must not overlap seq_lens");
  kvb::SelectParams prm{e.seq_lens, e.weights,    e.weight_stride, keep,    kept_lens, e.batch,
                        e.kv_heads, e.max_tokens, e.budget,        e.sinks, e.recent};
  // CTAs a segment: one for every 2,048 tokens, at most the eight of a
  // portable cluster (sixteen: selecting and moving 8,192 of 65,536 tokens 73 us
  // for 51), and no more than fill the SMs twice (16 x 16K tokens on 8 heads: 90
  // us in clusters of eight, whose shared histograms queue).
  uint32_t ctas = 1;
  while (ctas < 8 && uint64_t(ctas) * 2048 < e.max_tokens &&
         uint64_t(e.batch) * e.kv_heads * ctas * 2 <= uint64_t(2 * detail::device_sms()))
    ctas *= 2;
  const uint32_t part = (e.max_tokens + ctas - 1) / ctas;
  const uint32_t smem = std::min(part, kvb::kSelectKeys) * uint32_t(sizeof(uint32_t));
  const Kv4Kernel k{reinterpret_cast<const void*>(&kvb::select_tokens_kernel), kvb::kSelectKeys * uint32_t(sizeof(uint32_t))};
  resident_ctas(k, kvb::kSelectThreads);
  void* args[] = {&prm};
  g_launched.store(true, std::memory_order_relaxed);
  detail::launch_kernel_cluster(k.fn, dim3(e.batch * e.kv_heads * ctas), dim3(kvb::kSelectThreads), ctas, smem, stream, args,
                                "token selection launch");
}

void compact_kv4(const Kv4Pool& pool, const Kv4Eviction& e, const uint32_t* block_table,
                 uint32_t table_stride, const int32_t* keep, const uint32_t* new_table,
                 uint32_t new_stride, float* new_weights, int64_t new_weight_stride,
                 cudaStream_t stream) {
  check_pool(pool);
  check_eviction(e);
  if (e.kv_heads != pool.kv_heads) throw std::invalid_argument("eviction kv_heads differ from the pool's");
  if (!block_table || !keep || !new_table)
    throw std::invalid_argument("block_table, keep and new_table must be non-null");
  if (!aligned_to(block_table, 4) || !aligned_to(keep, 4) || !aligned_to(new_table, 4) ||
      !aligned_to(new_weights, 4))
    throw std::invalid_argument("eviction buffers must be 4-byte aligned");
  if (table_stride == 0 || new_stride == 0)
    throw std::invalid_argument("block-table strides must be positive");
  if (uint64_t(std::min(e.budget, e.max_tokens)) > uint64_t(new_stride) * pool.page_tokens)
    throw std::invalid_argument("budget exceeds the new block-table row capacity");
  if (new_weights != nullptr && new_weight_stride < int64_t(e.budget))
    throw std::invalid_argument("new_weight_stride must be at least budget");
  // CTAs write the new rows while others read the old ones.
  if (new_weights != nullptr && rows_overlap(e.weights, e.weight_stride, e.max_tokens, new_weights, new_weight_stride,
                                             e.budget, int64_t(e.batch) * e.kv_heads))
    throw std::invalid_argument("new_weights must not overlap weights");
  kvb::CompactParams prm{view(pool),   e.seq_lens,   e.weights,   e.weight_stride,   block_table,
                         keep,         new_table,    new_weights, new_weight_stride, e.batch,
                         e.max_tokens, e.budget,     table_stride, new_stride,       pool.page_tokens,
                         log2_page(pool)};
  const void* fn = by_dim(pool.dim, [&](auto d) {
    return reinterpret_cast<const void*>(&kvb::compact_kv4_kernel<decltype(d)::value>);
  });
  void* args[] = {&prm};
  launch_kernel_pdl(fn, dim3((e.budget + kvb::kCompactTile - 1) / kvb::kCompactTile, e.kv_heads, e.batch),
                    dim3(kvb::kCompactThreads), 0, stream, args, "kv4 compaction launch");
}

// ---------------------------------------------------------------------------

namespace detail {

cudaError_t read_kv4_status(int* status) noexcept {
  *status = 0;
  if (!g_launched.load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t code = cudaMemcpyFromSymbol(status, kvb::g_kvb_status, sizeof(int));
  if (code != cudaSuccess || *status == 0) return code;
  const int zero = 0;
  return cudaMemcpyToSymbol(kvb::g_kvb_status, &zero, sizeof(int));
}

}  // namespace detail

}  // namespace kvbridge
