#pragma once
// Attention over the 4-bit pool, and the attention weight that each cached
// token gets (include/kvbridge/attention_kv4.h).
//
// Schedule. The attended tokens of a sequence are runs of 64-token stages;
// one segment per (sequence, KV head, group of query columns). The segments'
// stages, concatenated, are cut into equal contiguous ranges, one per warp of
// about one full wave; a warp's part of a segment is a piece and gives one
// partial result, or the output itself where the piece is the whole segment.
// A windowed call leaves the stages between the prefix and the window out of
// the list, so they are never read.
//
// Warps share nothing: each has its own slot for K and for V (codes and
// params) and refills one with 16-byte asynchronous copies as soon as it has
// read it: the next K arrives while this stage's softmax and output run, the
// next V while the next scores do. No producer warp and no barriers. (One bulk
// copy per array and page instead of the eighteen 512-byte copy instructions
// of a stage left the warps queueing for the bulk-copy unit: 0.7 of 3.2 us a
// stage with 64-token pages, 2 of 5.6 us with 16-token pages.)
//
// Arithmetic (int8 tensor cores, exact s32 sums; codes 0..15 are int8
// operands after a mask or a shift and a mask, two values a byte):
//   scores   The query side is the A operand: each query value as three
//            signed base-256 digits of a fixed-point number, one A row per
//            (column, digit). x = scale_t * (A . (codes - 8)) + (lo_t + 8
//            scale_t) * sum(q) in fp32: the sums start at -8 * sum(digits),
//            so that little cancels between the two parts.
//   output   P = exp(x - m) * v_scale as unsigned fixed point against the
//            tile's largest, in base-256 digits that are the mantissa bytes
//            of P * 2^e + 2^23. These sums count codes from -8 too; the part
//            that carries lo, sum exp(x - m) * (lo + 8 v_scale), is in fp32.
//
// Column layouts: C query columns a segment (4 or 8) and PD digits of P.
//   q      Rows c and c + 8 of the first m16 tile are digits 0 and 1 of
//          column c; with 8 columns digit 2 is row c of a second tile, with 4
//          it is row c + 4 of the first.
//   P      8 columns: rows c and c + 8 are digits 0 and 1. 4 columns: lanes c
//          and c + 4 share a column and split its tokens (and the work on
//          them): rows c and c + 8 have the digits of one's tokens, rows c + 4
//          and c + 12 those of the other's, zeros for the rest; each lane
//          sums its own share of the output. PD = 3: digit 2 in the same rows
//          of a second tile.
// PD = 2 holds P * v_scale to 2^-16 of the tile's largest: a token's part of the
// output is off by at most 8 * 2^-16 of that, where its codes stand for values
// known to half of their step only (2^-1 of P * v_scale). One f16 sequence of
// 64K tokens ends 2.15e-4 from 64 bits, the exact result rounded to f16 2.12e-4;
// bf16 shows no difference. fp32 outputs take 3. Queries are held to 2^-22 of
// their row's largest, fp32 ones too, by the same argument against the keys'
// codes; the lse is fp32 always, hence three q digits for every type.
//
// Bound: 144 bytes a cached token and KV head at dim 128, and 4 * dim flops a
// token and query row. With four query columns a KV head the copies bound it:
// 32 sequences of 1K to 32K tokens (612 MB) take 106 us, 5.8 TB/s. With eight,
// or at dim 256 with digits for several rows, the instructions between the
// copies do (issue slots half used at twelve warps an SM, the rest waits for
// the warp's own chain of products and shuffles): 64 x 16K tokens with 16-token
// pages 249 us, 4.9 TB/s; eight rows of 24 heads of dim 256 over 32K tokens 60
// to 64 us, 0.1 PFLOP/s. Explicit positions mask every stage and are loaded
// within it: 16 x 16K tokens with 4 columns 75 us so, 59 us by index. Short calls
// are bound by latency: one sequence of 4,096 tokens takes 11.0 us, of which the
// two kernels' starts and the merge are about 7.
#include "kv4_common.cuh"
#include "kvb_schedule.h"

namespace kvb {

constexpr int kv4_q_tiles(int cols) { return cols == 4 ? 1 : 2; }       // m16 tiles of the scores
constexpr int kv4_p_tiles(int digits) { return digits == 3 ? 2 : 1; }   // and of the output
constexpr int kv4_tokens(int cols) { return cols == 4 ? 8 : 16; }       // of a stage, a lane

// What a kernel knows of the score rule: causal by index alone; also window
// and prefix by index; or everything (cap, bias, explicit positions).
enum : int { kRulesNone = 0, kRulesMask = 1, kRulesAll = 2 };

constexpr int kKv4Warps = 4;
constexpr int kKv4Threads = 32 * kKv4Warps;
constexpr uint32_t kNoUnit = 0xffffffffu;

struct Kv4AttendParams {
  Kv4View pool;
  Kv4Rule rule;
  const void* q;
  int64_t batch_stride, row_stride;
  const uint32_t* seq_lens;
  const uint32_t* table;
  uint32_t batch, rows, q_heads, group, table_stride, max_tokens;
  uint32_t page_tokens, log2_page;
  uint32_t col_groups;  // groups of query columns (rows * group) of a KV head
  uint32_t workers;     // warps of the grid
  int32_t type;   // of q and out: 0 f32, 1 f16, 2 bf16
  bool vector_q;  // 16-byte aligned query rows
  bool direct;    // one warp per segment, nothing to merge
  // Partials of piece (warp w, segment i) in slot w + i: per column D sums and
  // {max, sum}; the first and last warp of every segment.
  float* part;
  float2* part_ml;
  uint2* seg_warps;
  void* out;
  float* lse;
  // accumulate_weights_kv4
  const float* lse_in;
  float* weights;
  int64_t weight_stride;
};

// ---------------------------------------------------------------------------
// The stage list.

// A segment being walked; positions are relative to the warp's first stage.
struct Kv4Cursor {
  uint32_t b, seg;
  uint32_t len;     // tokens of sequence b
  uint32_t stages;  // of the segment
  uint32_t head, skip;  // stage j of the segment is j (j < head) or j + skip
  int32_t base;     // where the segment's stage 0 lies
};

// HINT: read before the wait for the preceding kernel, past L1; such values
// only steer prefetches, or are compared with what the wait lets through.
template <int RULES, bool HINT = false>
__device__ __forceinline__ void kv4_load_sequence(const Kv4AttendParams& p, Kv4Cursor& c) {
  const uint32_t len = HINT ? __ldcg(p.seq_lens + c.b) : kv4_load(p.seq_lens + c.b);
  c.len = min(len, p.max_tokens);
  c.stages = (c.len + kStageTokens - 1) / kStageTokens;
  c.head = c.stages;
  c.skip = 0;
  if (RULES != kRulesNone && p.rule.window != 0 && p.pool.pos == nullptr && p.rule.q_pos == nullptr) {
    // The first row's window starts at len - rows - window + 1.
    const uint64_t reach = uint64_t(p.rows) + p.rule.window - 1;
    const uint32_t from = reach < c.len ? uint32_t(c.len - reach) / kStageTokens : 0u;
    int32_t fix = 0;
    if (p.rule.prefix != nullptr) fix = int32_t(HINT ? __ldcg(p.rule.prefix + c.b) : kv4_load(p.rule.prefix + c.b));
    c.head = (uint32_t(max(0, min(fix, int32_t(c.len)))) + kStageTokens - 1) / kStageTokens;
    if (c.head < from) {
      c.skip = from - c.head;
      c.stages -= c.skip;
    }
  }
}

template <int RULES>
__device__ __forceinline__ uint32_t kv4_stage_count(const Kv4AttendParams& p, uint32_t b) {
  Kv4Cursor c;
  c.b = b;
  kv4_load_sequence<RULES>(p, c);
  return c.stages;
}

// The next segment that has stages (b = batch at the end).
template <int RULES>
__device__ __forceinline__ void kv4_next_segment(const Kv4AttendParams& p, uint32_t segs, Kv4Cursor& c) {
  c.base += int32_t(c.stages);
  if (++c.seg < segs) return;
  c.seg = 0;
  while (++c.b < p.batch) {
    kv4_load_sequence<RULES>(p, c);
    if (c.stages != 0) return;
  }
}

// Equal ranges of the `total` stages, the first ones a stage longer. (A 64-bit
// division is a few hundred instructions on the path to the first copy.)
__device__ __forceinline__ uint32_t kv4_range(uint64_t total, uint32_t workers, uint32_t w, uint64_t& first) {
  workers = uint32_t(min(uint64_t(workers), total));
  if (w >= workers) return 0;
  const uint64_t each = total >> 32 ? total / workers : uint32_t(total) / workers;
  const uint32_t more = uint32_t(total - each * workers);
  first = w * each + min(w, more);
  return uint32_t(each) + (w < more ? 1u : 0u);
}

// `into`: the first stage, counted from the sequence's first.
__device__ __forceinline__ void kv4_enter(uint64_t into, Kv4Cursor& c) {
  c.seg = into >> 32 ? uint32_t(into / c.stages) : uint32_t(into) / c.stages;
  c.base = -int32_t(into - uint64_t(c.seg) * c.stages);
}

// Up to 32 sequences, lane b holding sequence b in `own`: the range of worker
// w and the cursor at its first stage. Returns its number of stages.
//
// A worker that meets the start of a segment prepares another query and writes
// another partial, about a stage's time: where ranges are long enough, every
// segment counts one stage more than it has, before its first. (16 sequences
// of 4,200 seen tokens with two rows each ended 6 us after the median warp.)
__device__ __forceinline__ uint32_t kv4_locate_lanes(const Kv4AttendParams& p, uint32_t w, uint32_t segs,
                                                     const Kv4Cursor& own, Kv4Cursor& c) {
  const uint32_t lane = threadIdx.x & 31, mine = lane < p.batch ? own.stages : 0u;
  uint64_t real = mine;  // stages of a head up to and with this sequence
  uint32_t held = mine != 0 ? 1u : 0u;  // sequences that have any
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, real, o);
    const uint32_t z = __shfl_up_sync(0xffffffffu, held, o);
    if (lane >= uint32_t(o)) real += y, held += z;
  }
  const uint64_t all = __shfl_sync(0xffffffffu, real, 31) * segs;
  // (with two counted stages or more a range has one that is real)
  const uint32_t extra = all >= uint64_t(4) * p.workers ? 1u : 0u;
  const uint64_t counted = real + uint64_t(held) * extra;
  const uint64_t total = __shfl_sync(0xffffffffu, counted, 31) * segs;
  uint64_t first = 0;
  const uint32_t length = kv4_range(total, p.workers, w, first);
  if (length == 0) return 0;
  // Real stages before counted stage x, and where x is.
  auto enter = [&](uint64_t x, Kv4Cursor& at, uint32_t& j) {
    const int b = __ffs(__ballot_sync(0xffffffffu, counted * segs > x)) - 1;
    at.b = b;
    at.stages = __shfl_sync(0xffffffffu, mine, b);
    const uint64_t into = x - (__shfl_sync(0xffffffffu, counted, b) - at.stages - extra) * segs;
    const uint32_t each = at.stages + extra;
    at.seg = into >> 32 ? uint32_t(into / each) : uint32_t(into) / each;
    const uint32_t off = uint32_t(into - uint64_t(at.seg) * each);
    j = off > extra ? off - extra : 0u;
    return (__shfl_sync(0xffffffffu, real, b) - at.stages) * segs + uint64_t(at.seg) * at.stages + j;
  };
  uint32_t j;
  const uint64_t from = enter(first, c, j);
  c.base = -int32_t(j);
  c.len = __shfl_sync(0xffffffffu, own.len, c.b);
  c.head = __shfl_sync(0xffffffffu, own.head, c.b);
  c.skip = __shfl_sync(0xffffffffu, own.skip, c.b);
  uint64_t to = all;
  Kv4Cursor end;
  if (first + length < total) to = enter(first + length, end, j);
  return uint32_t(to - from);
}

// The same for more sequences, or for a direct call (worker w = segment w).
template <int RULES>
__device__ uint32_t kv4_locate(const Kv4AttendParams& p, uint32_t w, uint32_t segs, Kv4Cursor& c) {
  const uint32_t lane = threadIdx.x & 31;
  if (p.direct) {
    if (w >= p.workers) return 0;
    c.b = w / segs;
    c.seg = w % segs;
    c.base = 0;
    kv4_load_sequence<RULES>(p, c);
    return c.stages;
  }
  uint64_t total = 0;
  for (uint32_t b = lane; b < p.batch; b += 32) total += kv4_stage_count<RULES>(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  uint64_t first = 0, before = 0;
  const uint32_t count = kv4_range(total * segs, p.workers, w, first);
  if (count == 0) return 0;
  for (uint32_t from = 0; from < p.batch; from += 32) {
    const uint32_t n = from + lane < p.batch ? kv4_stage_count<RULES>(p, from + lane) : 0u;
    uint64_t upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= uint32_t(o)) upto += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, (before + upto) * segs > first);
    if (hit != 0) {
      const int at = __ffs(hit) - 1;
      before = (before + __shfl_sync(0xffffffffu, upto - n, at)) * segs;
      c.b = from + at;
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  kv4_load_sequence<RULES>(p, c);
  kv4_enter(first - before, c);
  return count;
}

// Finds the warp's range around the wait for the preceding kernel. Up to 32
// sequences are located before it, from lengths that are only taken if they
// are the same after it; the first stage's pages, the next one's table entries
// and the query rows are prefetched into L2 meanwhile.
template <int D, bool V, int RULES>
__device__ __forceinline__ uint32_t kv4_start(const Kv4AttendParams& p, uint32_t w, uint32_t segs, uint32_t cols,
                                              Kv4Cursor& c) {
  const uint32_t lane = threadIdx.x & 31;
  if (p.direct || p.batch > 32) {
    grid_launch_dependents();
    grid_dependency_wait();
    return kv4_locate<RULES>(p, w, segs, c);
  }
  Kv4Cursor hint;
  hint.b = min(lane, p.batch - 1);
  kv4_load_sequence<RULES, true>(p, hint);
  uint32_t count = kv4_locate_lanes(p, w, segs, hint, c);
  if (count != 0) {
    const uint32_t j = uint32_t(-c.base), stage = RULES && j >= c.head ? j + c.skip : j;
    const uint32_t page = (stage * kStageTokens + 16 * (lane & 3)) >> p.log2_page;
    const uint32_t* entry = p.table + size_t(c.b) * p.table_stride + page;
    const uint32_t phys = (page << p.log2_page) < c.len ? __ldcg(entry) : kNoUnit;
    const uint32_t h = c.seg / p.col_groups, part = lane >> 2;
    const bool pages = (lane & 3) < (kStageTokens >> p.log2_page) && part < (V ? 4 : 2);
    // Lane q + 4 part: array `part` of page q of the stage (with 16-token
    // pages lane q has page q; with larger ones the first lanes').
    const uint32_t mine = __shfl_sync(0xffffffffu, phys, (lane & 3) << (p.log2_page - 4));
    if (pages && mine < p.pool.pages) {
      const size_t unit = size_t(mine) * p.pool.kv_heads + h;
      const uint32_t P = p.page_tokens;
      if (part == 0) prefetch_l2(p.pool.k + unit * P * (D / 2), P * (D / 2));
      if (part == 1) prefetch_l2(p.pool.kp + unit * P, P * 8);
      if (part == 2) prefetch_l2(p.pool.v + unit * P * (D / 2), P * (D / 2));
      if (part == 3) prefetch_l2(p.pool.vp + unit * P, P * 8);
    }
    const uint32_t col = (c.seg % p.col_groups) * cols + (lane >> 2) % cols;
    if (col < p.rows * p.group) {
      const int64_t at = int64_t(c.b) * p.batch_stride + int64_t(col / p.group) * p.row_stride +
                         int64_t(h * p.group + col % p.group) * D + (D / 4) * (lane & 3);
      prefetch_line_l2(static_cast<const uint8_t*>(p.q) + at * (p.type == 0 ? 4 : 2));
    }
  }
  grid_launch_dependents();
  grid_dependency_wait();
  Kv4Cursor own;
  own.b = hint.b;
  kv4_load_sequence<RULES>(p, own);
  if (!__all_sync(0xffffffffu, own.len == hint.len && own.stages == hint.stages && own.head == hint.head &&
                                   own.skip == hint.skip))
    count = kv4_locate_lanes(p, w, segs, own, c);
  return count;
}

// ---------------------------------------------------------------------------
// One warp's slots.

// K codes, K params, V codes (pages of 16 and 32 tokens 32 and 64 bytes
// further apart), V params. The params of 16 tokens are 144 bytes apart. With
// these gaps a quarter-warp's reads of four token groups or several pages hit
// different banks. V false: K alone.
constexpr uint32_t kKv4ParamPitch = 144;
// {scale, lo} in the slots of 16 tokens whose page is not in the pool: no row
// has a negative scale. Attention's K is NaN instead, which no maximum takes.
constexpr float kKv4Absent = -1.0f;
template <int D, bool V>
struct Kv4Smem {
  static constexpr uint32_t kCodes = kStageTokens * D / 2;
  static constexpr uint32_t kParams = kStageTokens / 16 * kKv4ParamPitch;
  static constexpr uint32_t kOffKp = kCodes;
  static constexpr uint32_t kOffV = kOffKp + kParams;
  static constexpr uint32_t kOffVp = kOffV + kCodes + 128;
  static constexpr uint32_t kWarp = V ? kOffVp + kParams : kOffV;
  static constexpr uint32_t kBytes = kKv4Warps * kWarp;
};

__device__ __forceinline__ uint32_t kv4_v_pitch(uint32_t page_bytes, uint32_t P) {
  return P == 64 ? page_bytes : page_bytes + 2 * P;
}

template <int D, bool V, int RULES>
struct Kv4Feeder {
  uint8_t* slots;
  uint32_t addr;   // of slots, in shared memory
  Kv4Cursor cur;   // the segment of the next stage to look up
  uint32_t next;   // that stage, relative to the warp's first
  uint32_t count;  // stages of the warp
  uint32_t segs;
  // The page of the stage's 16-token group lane % 4, looked up last: in
  // flight until it is used.
  uint32_t phys, head;

  __device__ void init(uint8_t* smem, uint32_t warp) {
    slots = smem + warp * Kv4Smem<D, V>::kWarp;
    addr = smem_addr(slots);
  }

  // The block-table entry of the lane's 16-token group of stage `at`.
  __device__ __forceinline__ uint32_t entry_of(const Kv4AttendParams& p, uint32_t at) const {
    const uint32_t j = uint32_t(int32_t(at) - cur.base);
    const uint32_t stage = RULES && j >= cur.head ? j + cur.skip : j;
    return (stage * kStageTokens + 16 * (threadIdx.x & 3)) >> p.log2_page;
  }

  // Starts the lookup of the pages of stage `next`; kNoUnit where there is none.
  __device__ __forceinline__ void lookup(const Kv4AttendParams& p) {
    phys = kNoUnit;
    if (next < count) {
      while (int32_t(next) >= cur.base + int32_t(cur.stages)) kv4_next_segment<RULES>(p, segs, cur);
      head = p.col_groups == 1 ? cur.seg : cur.seg / p.col_groups;
      const uint32_t page = entry_of(p, next);  // all of it: V's quarters are not tokens
      if ((page << p.log2_page) < cur.len) phys = kv4_load(p.table + size_t(cur.b) * p.table_stride + page);
      ++next;
    }
  }

  // Starts the copies of the K or the V of the stage looked up last. 64-token
  // pages: every lane has looked up the same page.
  template <bool OF_V>
  __device__ __forceinline__ void copy_page(const Kv4AttendParams& p) {
    using S = Kv4Smem<D, V>;
    const uint32_t lane = threadIdx.x & 31;
    const size_t unit = size_t(phys) * p.pool.kv_heads + head;
    const uint8_t* src = (OF_V ? p.pool.v : p.pool.k) + unit * (32 * D) + 16 * lane;
    const uint32_t dst = addr + (OF_V ? S::kOffV : 0u) + 16 * lane;
#pragma unroll
    for (uint32_t i = 0; i < D / 16; ++i) copy16_async(dst + 512 * i, src + 512 * i);
    copy16_async(addr + (OF_V ? S::kOffVp : S::kOffKp) + (lane >> 3) * kKv4ParamPitch + (lane & 7) * 16,
                 reinterpret_cast<const uint8_t*>((OF_V ? p.pool.vp : p.pool.kp) + unit * 64 + 2 * lane));
  }

  // Smaller pages: a quarter of the stage (of its 2 or 4 pages' codes) at a
  // time, from the unit that lane g has looked up.
  template <bool OF_V, bool ALL>
  __device__ __forceinline__ void copy_groups(const Kv4AttendParams& p, uint32_t unit) {
    using S = Kv4Smem<D, V>;
    const uint32_t lane = threadIdx.x & 31, log2_page = p.log2_page;
    const uint32_t page_bytes = (D / 2) << log2_page, in_page = p.page_tokens - 1;
    const uint8_t* codes = (OF_V ? p.pool.v : p.pool.k) + 16 * lane;
    const uint32_t dst = addr + (OF_V ? S::kOffV : 0u) + 16 * lane;
    const uint32_t gap = OF_V ? kv4_v_pitch(page_bytes, p.page_tokens) - page_bytes : 0u;
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g) {
      const uint32_t u = __shfl_sync(0xffffffffu, unit, g);
      const uint8_t* src = codes + size_t(u) * page_bytes + (16 * g & in_page) * (D / 2);
      if (ALL || u != kNoUnit)
#pragma unroll
        for (uint32_t i = 0; i < D / 64; ++i)
          copy16_async(dst + g * (8 * D) + 512 * i + ((16 * g) >> log2_page) * gap, src + 512 * i);
    }
    // Tokens 2 lane and 2 lane + 1 of group lane / 8.
    const uint32_t u = __shfl_sync(0xffffffffu, unit, lane >> 3);
    if (ALL || u != kNoUnit)
      copy16_async(addr + (OF_V ? S::kOffVp : S::kOffKp) + (lane >> 3) * kKv4ParamPitch + (lane & 7) * 16,
                   reinterpret_cast<const uint8_t*>((OF_V ? p.pool.vp : p.pool.kp) + (size_t(u) << log2_page) +
                                                    (2 * lane & in_page)));
  }

  // The lane's group of the stage is absent: two of its tokens a lane.
  template <bool OF_V>
  __device__ __forceinline__ void mark_absent() {
    using S = Kv4Smem<D, V>;
    const uint32_t lane = threadIdx.x & 31;
    const float scale = V && !OF_V ? __int_as_float(0x7fffffff) : kKv4Absent;
    *reinterpret_cast<float4*>(slots + (OF_V ? S::kOffVp : S::kOffKp) + (lane & 3) * kKv4ParamPitch + (lane >> 2) * 16) =
        make_float4(scale, 0.f, scale, 0.f);
  }

  template <bool OF_V>
  __device__ __forceinline__ void copy(const Kv4AttendParams& p) {
    const bool ok = phys < p.pool.pages;
    // A bad id, which may have kNoUnit's value; not a group past the sequence's end.
    if (!ok && (entry_of(p, next - 1) << p.log2_page) < cur.len) {
      if (!OF_V) atomicMax(&g_kvb_status, kKv4BadPage);
      mark_absent<OF_V>();
    }
    if (p.log2_page == 6) {
      if (ok) copy_page<OF_V>(p);
    } else {
      const uint32_t unit = ok ? phys * p.pool.kv_heads + head : kNoUnit;
      if (__all_sync(0xffffffffu, ok))
        copy_groups<OF_V, true>(p, unit);
      else
        copy_groups<OF_V, false>(p, unit);
    }
    copy_commit();
  }
};

// ---------------------------------------------------------------------------
// Queries.

__device__ __forceinline__ void kv4_half_pair(uint32_t w, bool bf16, float& a, float& b) {
  if (bf16) {
    a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x, b = f.y;
  }
}

// Eight values of each word of a lane's part of a query row, as they lie in
// memory: loads in flight until they are used. Rows that are not 16-byte
// aligned are read where the values are wanted.
template <int D>
struct Kv4RawQuery {
  uint4 w[D / 32][2];  // 16-bit values: the first alone
};

// The A operand of the scores for one group of columns. Lane (grp, tig) =
// (lane / 4, lane % 4) holds column grp (4 columns: grp % 4) at the dims of its
// quarter of each K row: word i of the lane's packed row covers 8 dims, the
// even ones in the low halves (a[.][0], a[.][1]), the odd ones in the high
// halves (a[.][2], a[.][3]).
template <int D, int C>
struct Kv4Query {
  uint32_t a[kv4_q_tiles(C)][D / 32][4];
  int start[kv4_q_tiles(C)][2];  // -8 * digit sums of rows grp and grp + 8
  // score = scale_t * (A . (codes - 8)) + (lo_t + 8 scale_t) * sum, the dot
  // product in parts: 8 columns digits 0 and 1, digit 2; 4 columns the
  // lane's own digits, the other lane's.
  float own, other, sum;
  float slope;
  int32_t pos;     // query position
};

// First dim of word i of the lane's part of a packed row.
template <int D>
__device__ __forceinline__ uint32_t kv4_word_dim(uint32_t tig, uint32_t i) {
  if constexpr (D == 256) return 128 * (i / 4) + 32 * tig + 8 * (i % 4);
  return (D / 4) * tig + 8 * i;
}

// Where a lane's column of a segment is: the query row's first element.
template <int D, int C>
__device__ __forceinline__ bool kv4_query_at(const Kv4AttendParams& p, uint32_t b, uint32_t h, uint32_t col_group,
                                             uint32_t& r, uint32_t& head, int64_t& at) {
  const uint32_t col = col_group * C + ((threadIdx.x & 31) >> 2) % C;
  const bool valid = col < p.rows * p.group;
  r = valid ? col / p.group : 0;
  head = h * p.group + (valid ? col % p.group : 0);
  at = int64_t(b) * p.batch_stride + int64_t(r) * p.row_stride + int64_t(head) * D;
  return valid;
}

template <int D, int C>
__device__ __forceinline__ void kv4_fetch_query(const Kv4AttendParams& p, uint32_t b, uint32_t h, uint32_t col_group,
                                                Kv4RawQuery<D>& raw) {
  if (!p.vector_q) return;
  uint32_t r, head;
  int64_t at;
  kv4_query_at<D, C>(p, b, h, col_group, r, head, at);
  const int bytes = p.type == 0 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.q) +
                                                      (at + kv4_word_dim<D>(threadIdx.x & 3, i)) * bytes);
    raw.w[i][0] = kv4_load(src);
    if (p.type == 0) raw.w[i][1] = kv4_load(src + 1);
  }
}

template <int D, int C, int RULES>
__device__ void kv4_make_query(const Kv4AttendParams& p, uint32_t b, uint32_t h, uint32_t col_group, uint32_t len,
                               const Kv4RawQuery<D>& raw, Kv4Query<D, C>& qf) {
  const uint32_t lane = threadIdx.x & 31, grp = lane >> 2, tig = lane & 3;
  uint32_t r, head;
  int64_t at;
  const bool valid = kv4_query_at<D, C>(p, b, h, col_group, r, head, at);
  float v[D / 32][8];
  if (!p.vector_q) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t x = at + kv4_word_dim<D>(tig, i) + e;
        float unused;
        if (p.type == 0) v[i][e] = kv4_load(static_cast<const float*>(p.q) + x);
        else kv4_half_pair(kv4_load(static_cast<const uint16_t*>(p.q) + x), p.type == 2, v[i][e], unused);
      }
  } else if (p.type == 0) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 w = raw.w[i][k];
        v[i][4 * k] = __uint_as_float(w.x), v[i][4 * k + 1] = __uint_as_float(w.y);
        v[i][4 * k + 2] = __uint_as_float(w.z), v[i][4 * k + 3] = __uint_as_float(w.w);
      }
  } else {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const uint4 w = raw.w[i][0];
      kv4_half_pair(w.x, p.type == 2, v[i][0], v[i][1]);
      kv4_half_pair(w.y, p.type == 2, v[i][2], v[i][3]);
      kv4_half_pair(w.z, p.type == 2, v[i][4], v[i][5]);
      kv4_half_pair(w.w, p.type == 2, v[i][6], v[i][7]);
    }
  }
  float amax = 0.f;  // NaN if a value is
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 8; e += 2) amax = max3_abs_nan(amax, v[i][e], v[i][e + 1]);
  amax = max3_abs_nan(amax, amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = max3_abs_nan(amax, amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  // Fixed point n = rint(q * up), |n| <= 2^22: n = d0 + 256 d1 + 65536 d2
  // with signed digits; up is a power of two.
  int e = int((__float_as_uint(amax) >> 23) & 0xffu) - 126;  // amax < 2^e
  e = max(-100, min(128, e));
  const float up = __uint_as_float(uint32_t(127 + 22 - e) << 23);
  const float down = __uint_as_float(uint32_t(127 + e - 22) << 23);
  // fma(q, up, 1.5 * 2^23) rounds to the integer in the low mantissa bits;
  // removing the sum's bias and adding 0x808080 leaves n + 0x808080, whose
  // bytes are the digits + 128.
  constexpr float kRoundInt = 12582912.0f;
  constexpr uint32_t kBias = 0x808080u - 0x4B400000u;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      uint32_t w[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) w[x] = valid ? __float_as_uint(fmaf(v[i][2 * x + odd], up, kRoundInt)) + kBias : 0x808080u;
      const uint32_t x = __byte_perm(w[0], w[1], 0x5140), y = __byte_perm(w[2], w[3], 0x5140);
      const uint32_t d0 = __byte_perm(x, y, 0x5410) ^ 0x80808080u, d1 = __byte_perm(x, y, 0x7632) ^ 0x80808080u;
      const uint32_t x2 = __byte_perm(w[0], w[1], 0x0062), y2 = __byte_perm(w[2], w[3], 0x0062);
      const uint32_t d2 = __byte_perm(x2, y2, 0x5410) ^ 0x80808080u;
      if constexpr (C == 4) {
        qf.a[0][i][2 * odd] = grp >= 4 ? d2 : d0;
        qf.a[0][i][2 * odd + 1] = grp >= 4 ? 0u : d1;
      } else {
        qf.a[0][i][2 * odd] = d0;
        qf.a[0][i][2 * odd + 1] = d1;
        qf.a[1][i][2 * odd] = d2;
        qf.a[1][i][2 * odd + 1] = 0u;
      }
    }
  int digits[kv4_q_tiles(C)][2];  // digit sums of rows grp and grp + 8
#pragma unroll
  for (int m = 0; m < kv4_q_tiles(C); ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      int s = 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        s = __dp4a(int(qf.a[m][i][r]), 0x01010101, s);
        s = __dp4a(int(qf.a[m][i][2 + r]), 0x01010101, s);
      }
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
      digits[m][r] = s;
      qf.start[m][r] = -8 * s;
    }
  // sum of n, exact: 256 values of at most 2^22, so at most 2^30 (and -8 times
  // that would not fit).
  int total = digits[0][0] + 256 * digits[0][1];
  if constexpr (C == 8) {
    total += 65536 * digits[1][0];
  } else {
    const int other = __shfl_xor_sync(0xffffffffu, total, 16);  // the upper lane has digit 2
    total = grp >= 4 ? 65536 * total + other : total + 65536 * other;
  }
  // Scores in log2 units, or in natural ones where a cap or a bias comes after.
  const float unit = RULES == kRulesAll ? p.rule.scale : p.rule.scale * kLog2e;
  const float dot = amax <= 3.402823466e38f ? down * unit : __int_as_float(0x7fffffff);
  qf.own = C == 4 && grp >= 4 ? 65536.f * dot : dot;
  qf.other = C == 4 && grp >= 4 ? dot : 65536.f * dot;
  qf.sum = float(total) * dot;
  qf.slope = RULES == kRulesAll && p.rule.slopes != nullptr ? kv4_load(p.rule.slopes + head) : 0.f;
  qf.pos = valid ? kv4_query_position(p.rule, b, r, p.rows, len) : -1;
}

// ---------------------------------------------------------------------------
// Dot products of one stage's tokens with the thread's column. N-tile j takes
// tokens 16 (n / 2) + 2 j + n % 2, so that a thread's C fragments (n = 2 tig,
// 2 tig + 1) are tokens 16 tig + 2 j and the next, and a quarter-warp reads
// two neighbouring K rows. 8 columns: sc[u] is token 16 tig + u. 4 columns:
// lane c keeps tokens 0-3 and 8-11 of the 16 (u = 0..7), lane c + 4 the rest.
__device__ __forceinline__ uint32_t kv4_token(int cols, int u) { return cols == 4 ? (u & 3) + 8 * (u >> 2) : u; }
template <int C>
__device__ __forceinline__ uint32_t kv4_first_token() {
  const uint32_t lane = threadIdx.x & 31;
  return 16 * (lane & 3) + (C == 4 ? 4 * (lane >> 4) : 0);
}

// Where the params of the thread's first token lie in a slot.
template <int C>
__device__ __forceinline__ uint32_t kv4_params_at() {
  const uint32_t t = kv4_first_token<C>();
  return (t >> 4) * kKv4ParamPitch + (t & 15) * 8;
}

template <int D, int C>
__device__ __forceinline__ void kv4_dots(const uint8_t* codes, const Kv4Query<D, C>& qf, float (&sc)[kv4_tokens(C)]) {
  const uint32_t lane = threadIdx.x & 31, grp = lane >> 2, tig = lane & 3;
  constexpr int kWords = D / 32;
  float part[C == 4 ? 16 : 1];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint8_t* row = codes + (16 * (grp >> 1) + 2 * j + (grp & 1)) * (D / 2);
    uint32_t w[kWords];
    if constexpr (D == 64) {
      const uint2 x = *reinterpret_cast<const uint2*>(row + 8 * tig);
      w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
      for (int c = 0; c < D / 128; ++c) {
        const uint4 x = *reinterpret_cast<const uint4*>(row + 64 * c + 16 * tig);
        w[4 * c] = x.x, w[4 * c + 1] = x.y, w[4 * c + 2] = x.z, w[4 * c + 3] = x.w;
      }
    }
    int acc[kv4_q_tiles(C)][4];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const uint32_t lo = w[i] & 0x0f0f0f0fu, hi = (w[i] >> 4) & 0x0f0f0f0fu;
#pragma unroll
      for (int m = 0; m < kv4_q_tiles(C); ++m) {
        const uint32_t* a = qf.a[m][i];
        const int s0 = qf.start[m][0], s1 = qf.start[m][1];
        if (i == 0)
          imma_16832(acc[m], a[0], a[1], a[2], a[3], lo, hi, s0, s0, s1, s1);
        else
          imma_16832(acc[m], a[0], a[1], a[2], a[3], lo, hi);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      // |digit dot| <= 128 * 8 * 256: exact in s32 with its neighbour
      const float x = float(acc[0][e] + 256 * acc[0][2 + e]);
      if constexpr (C == 8) sc[2 * j + e] = fmaf(x, qf.own, float(acc[1][e]) * qf.other);
      else part[2 * j + e] = x;
    }
  }
  if constexpr (C == 4) {
    // Lane c has digits 0 and 1 of all 16 tokens, lane c + 4 digit 2: swap.
    const bool upper = lane >= 16;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int t = kv4_token(4, u);
      const float give = upper ? part[t] : part[t + 4], keep = upper ? part[t + 4] : part[t];
      sc[u] = fmaf(keep, qf.own, __shfl_xor_sync(0xffffffffu, give, 16) * qf.other);
    }
  }
}

// x = softcap * tanh(x / softcap): the series where |x / softcap| < 0.3, which
// is all of most stages, else 1 - 2 / (e^2y + 1), which cancels near 0.
template <int N>
__device__ __forceinline__ void kv4_cap(float cap, float (&x)[N]) {
  const float inv = fminf(1.0f / cap, 3.402823466e38f);  // (a denormal cap's is infinite: 0 * inf)
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(x[i]));  // (a NaN takes either way)
  const bool far = __any_sync(0xffffffffu, top * inv >= 0.3f);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = x[i] * inv, y2 = y * y;
    float s = fmaf(y2, 62.0f / 2835.0f, -17.0f / 315.0f);
    s = fmaf(s, y2, 2.0f / 15.0f);
    s = fmaf(s, y2, -1.0f / 3.0f);
    const float near = fmaf(x[i], s * y2, x[i]);
    if (far) {
      const float u = fast_exp2(y * (2.0f * kLog2e));
      const float t = 1.0f - __fdividef(2.0f, u + 1.0f);
      x[i] = fabsf(y) < 0.3f ? near : cap * t;
    } else {
      x[i] = near;
    }
  }
}

// exp(x - y) of scores x and y: in natural units with kRulesAll (differences
// are small where the result is not), else in log2 units.
template <int RULES>
__device__ __forceinline__ float kv4_exp(float x, float y) {
  return fast_exp2(RULES == kRulesAll ? (x - y) * kLog2e : x - y);
}

// Which tokens of the stage at tb every query row sees, by their indices:
// those below the first row's position (and below the prefix), if they are
// within the last row's window. A warp-uniform test that spares most stages
// the masks. first, last: the rows' positions.
template <int RULES>
__device__ __forceinline__ bool kv4_all_visible(const Kv4AttendParams& p, uint32_t tb, uint32_t len, int32_t prefix) {
  const int32_t first = int32_t(len) - int32_t(p.rows), end = int32_t(tb + kStageTokens);
  if (RULES == kRulesNone) return end <= first + 1;
  if (RULES == kRulesAll && p.rule.q_pos != nullptr) return false;
  if (end <= min(prefix, int32_t(len))) return true;
  return end <= first + 1 && (p.rule.window == 0 || uint32_t(int32_t(len) - 1 - int32_t(tb)) < p.rule.window);
}

// Scores from the dot products; invisible ones -inf. Returns the thread's
// visible tokens as a bit mask. tb: the stage's first token; all: every token
// is visible; pos: the positions of the thread's quad's 16 tokens, or null for
// their indices.
template <int C, int RULES>
__device__ __forceinline__ uint32_t kv4_scores(const Kv4AttendParams& p, const uint8_t* params, uint32_t tb,
                                               uint32_t len, int32_t prefix, bool all, float sum, float slope,
                                               int32_t pq, const int32_t* pos, float (&sc)[kv4_tokens(C)]) {
  constexpr int kTokens = kv4_tokens(C);
  const uint32_t at = kv4_first_token<C>();
  const float4* par = reinterpret_cast<const float4*>(params + kv4_params_at<C>());
#pragma unroll
  for (int u = 0; u < kTokens; u += 2) {
    const float4 f = par[kv4_token(C, u) / 2];
    sc[u] = fmaf(sc[u], f.x, fmaf(8.f, f.x, f.y) * sum);
    sc[u + 1] = fmaf(sc[u + 1], f.z, fmaf(8.f, f.z, f.w) * sum);
  }
  const int32_t t0 = int32_t(tb + at);
  int32_t pk[RULES == kRulesAll ? kTokens : 1];
  if constexpr (RULES == kRulesAll) {
    if (p.rule.softcap > 0.f) kv4_cap(p.rule.softcap, sc);
    if (pos != nullptr) {
#pragma unroll
      for (int u = 0; u < kTokens; ++u) pk[u] = kv4_load(pos + (at & 15) + kv4_token(C, u));
    } else {
#pragma unroll
      for (int u = 0; u < kTokens; ++u) pk[u] = t0 + int32_t(kv4_token(C, u));
    }
    // Distances are exact in fp32 below 2^24. Positions of rows may be
    // negative: |pq - pk| as the larger minus the smaller.
    if (p.rule.slopes != nullptr) {
      if (pos != nullptr) {
#pragma unroll
        for (int u = 0; u < kTokens; ++u)
          sc[u] = fmaf(-slope, float(uint32_t(max(pq, pk[u])) - uint32_t(min(pq, pk[u]))), sc[u]);
      } else {
        const float away = float(int64_t(pq) - t0);
#pragma unroll
        for (int u = 0; u < kTokens; ++u) sc[u] = fmaf(-slope, fabsf(away - float(kv4_token(C, u))), sc[u]);
      }
    }
  }
  uint32_t seen = (1u << kTokens) - 1;
  if (!all) {
    seen = 0;
#pragma unroll
    for (int u = 0; u < kTokens; ++u) {
      const int32_t t = t0 + int32_t(kv4_token(C, u));
      bool on = t <= pq;  // pq < len
      if constexpr (RULES != kRulesNone)
        on = uint32_t(t) < len && kv4_visible(RULES == kRulesAll ? pk[u] : t, pq, p.rule.window, prefix);
      sc[u] = on ? sc[u] : -INFINITY;
      seen |= on ? 1u << u : 0u;
    }
  }
  return seen;
}

// ---------------------------------------------------------------------------
// Attention: one pass over a segment's stages with the running maximum m and
// the sums l = sum exp(x - m), o = sum exp(x - m) * v of every column.

template <int D>
struct Kv4State {
  float o[D / 16][4];  // dims 16 j + 4 tig + [0, 4) of the thread's column (or its share)
  float m;             // running max, the same in all lanes of a column
  float l, lo;         // the thread's part of sum p and of sum p * (lo + 8 scale)
};

template <int N>
__device__ __forceinline__ float kv4_max(const float (&x)[N]) {
  float y = x[0];
#pragma unroll
  for (int i = 1; i + 1 < N; i += 2) y = max3(y, x[i], x[i + 1]);
  return fmaxf(y, x[N - 1]);
}

template <int D, int C, int PD, int RULES, bool MASK>
__device__ __forceinline__ void kv4_softmax(const uint8_t* vparams, uint32_t seen, float (&sc)[kv4_tokens(C)],
                                            Kv4State<D>& st, uint32_t (&digit)[kv4_p_tiles(PD)][2][4],
                                            float& out_scale) {
  constexpr int kTokens = kv4_tokens(C);
  const bool upper = C == 4 && (threadIdx.x & 16) != 0;
  float top = kv4_max(sc);
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  if (C == 4) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
  const float m = fmaxf(st.m, top);
  const float sub = m == -INFINITY ? 0.f : m;
  const float alpha = m == st.m ? 1.f : kv4_exp<RULES>(st.m, sub);
  st.m = m;
  const float4* par = reinterpret_cast<const float4*>(vparams + kv4_params_at<C>());
  // Of a page that is not in the pool: the scores are NaN (or -inf), and the
  // maximum has passed over them.
  const bool absent = par[0].x == kKv4Absent;
  if (__any_sync(0xffffffffu, alpha != 1.f || absent)) {
    if (absent) {
#pragma unroll
      for (int u = 0; u < kTokens; ++u) sc[u] = -INFINITY;
    }
    st.l *= alpha;
    st.lo *= alpha;
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[j][e] *= alpha;
  }
#pragma unroll
  for (int u = 0; u < kTokens; u += 2) {
    const float4 f = par[kv4_token(C, u) / 2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float scale = e ? f.z : f.x, lo = e ? f.w : f.y;
      const float pr = kv4_exp<RULES>(sc[u + e], sub);
      st.l += pr;
      float w = pr * scale, mid = fmaf(8.f, scale, lo);
      if (MASK && !(seen >> (u + e) & 1u)) w = 0.f, mid = 0.f;  // whatever the slot holds
      st.lo = fmaf(mid, pr, st.lo);
      sc[u + e] = w;
    }
  }
  float big = kv4_max(sc);
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
  big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
  // Power of two (a little less, so that nothing rounds up to the next one)
  // that puts the tile's largest below 2^16 or 2^23: the fixed-point values
  // are the low bytes of sc * up + 2^23. (All tokens absent: big is -0 and the
  // digits are 0, whatever the scales.)
  constexpr uint32_t kTop = PD == 2 ? 269 : 276;
  constexpr float kLess = 1.0f - 1.0f / 16384.0f;
  const uint32_t ex = max(__float_as_uint(big) >> 23, kTop - 253u);
  const float up = kLess * __uint_as_float((kTop - ex) << 23);
  out_scale = (1.0f / kLess) * __uint_as_float((ex - (kTop - 254u)) << 23);
  // A fragments: tokens 8 i .. 8 i + 3 of the quad's 16 feed a[0] and a[1] of
  // fragment i, the next four a[2] and a[3].
#pragma unroll
  for (int h = 0; h < kTokens / 4; ++h) {
    uint32_t f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __float_as_uint(fmaf(sc[4 * h + e], up, 8388608.0f));
    const uint32_t x = __byte_perm(f[0], f[1], 0x5140), y = __byte_perm(f[2], f[3], 0x5140);
    uint32_t d[3] = {__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632), 0u};
    if constexpr (PD == 3)
      d[2] = __byte_perm(__byte_perm(f[0], f[1], 0x0062), __byte_perm(f[2], f[3], 0x0062), 0x5410);
#pragma unroll
    for (int k = 0; k < PD; ++k) {
      if constexpr (C == 4) {
        digit[k / 2][h][k % 2] = upper ? 0u : d[k];
        digit[k / 2][h][2 + k % 2] = upper ? d[k] : 0u;
      } else {
        digit[k / 2][h / 2][2 * (h % 2) + k % 2] = d[k];
      }
    }
  }
  if constexpr (PD == 3)
#pragma unroll
    for (int i = 0; i < 2; ++i) digit[1][i][1] = digit[1][i][3] = 0u;
}

// O += P . V for one stage. Thread (grp, tig) reads, for the dim pair 8 j +
// grp, the codes of its quad's 16 tokens; low halves are the even dims' tile,
// high halves (16 times the codes) the odd dims'.
template <int D, int PD>
__device__ __forceinline__ void kv4_output(const uint8_t* codes, uint32_t P, uint32_t pitch,
                                           const uint32_t (&digit)[kv4_p_tiles(PD)][2][4], float out_scale,
                                           Kv4State<D>& st) {
  const uint32_t lane = threadIdx.x & 31, grp = lane >> 2, tig = lane & 3;
  const uint8_t* base = codes + (16 * tig / P) * pitch + (16 * tig % P) + grp * P;
  const float odd_scale = out_scale * 0.0625f;
  // -8 * (sum of the row's digits), rows grp and grp + 8 of every tile: the
  // product with ones has it in every column.
  int start[kv4_p_tiles(PD)][2], start16[kv4_p_tiles(PD)][2];
#pragma unroll
  for (int m = 0; m < kv4_p_tiles(PD); ++m) {
    const uint32_t(&a)[2][4] = digit[m];
    constexpr uint32_t kOnes = 0x01010101u;
    int s[4];
    imma_u8_16832(s, a[0][0], a[0][1], a[0][2], a[0][3], kOnes, kOnes, 0, 0, 0, 0);
    imma_u8_16832(s, a[1][0], a[1][1], a[1][2], a[1][3], kOnes, kOnes, s[0], s[1], s[2], s[3]);
#pragma unroll
    for (int r = 0; r < 2; ++r) start[m][r] = -8 * s[2 * r], start16[m][r] = -128 * s[2 * r];
  }
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    const uint4 w = *reinterpret_cast<const uint4*>(base + 8 * j * P);
    int even[kv4_p_tiles(PD)][4], odd[kv4_p_tiles(PD)][4];
#pragma unroll
    for (int m = 0; m < kv4_p_tiles(PD); ++m) {
      const uint32_t(&a)[2][4] = digit[m];
      const int s0 = start[m][0], s1 = start[m][1], t0 = start16[m][0], t1 = start16[m][1];
      imma_u8_16832(even[m], a[0][0], a[0][1], a[0][2], a[0][3], w.x & 0x0f0f0f0fu, w.y & 0x0f0f0f0fu, s0, s0, s1, s1);
      imma_u8_16832(odd[m], a[0][0], a[0][1], a[0][2], a[0][3], w.x & 0xf0f0f0f0u, w.y & 0xf0f0f0f0u, t0, t0, t1, t1);
      imma_u8_16832(even[m], a[1][0], a[1][1], a[1][2], a[1][3], w.z & 0x0f0f0f0fu, w.w & 0x0f0f0f0fu, even[m][0],
                    even[m][1], even[m][2], even[m][3]);
      imma_u8_16832(odd[m], a[1][0], a[1][1], a[1][2], a[1][3], w.z & 0xf0f0f0f0u, w.w & 0xf0f0f0f0u, odd[m][0],
                    odd[m][1], odd[m][2], odd[m][3]);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      // exact: |sum| <= 255 * 128 * 64 a digit, times 257 below 2^30
      float x = float(even[0][e] + 256 * even[0][2 + e]), y = float(odd[0][e] + 256 * odd[0][2 + e]);
      if constexpr (PD == 3) {
        x = fmaf(float(even[1][e]), 65536.f, x);
        y = fmaf(float(odd[1][e]), 65536.f, y);
      }
      st.o[j][2 * e] = fmaf(x, out_scale, st.o[j][2 * e]);
      st.o[j][2 * e + 1] = fmaf(y, odd_scale, st.o[j][2 * e + 1]);
    }
  }
}

__device__ __forceinline__ void kv4_store_out(void* out, size_t at, int32_t type, float x) {
  if (type == 0) static_cast<float*>(out)[at] = x;
  else if (type == 1) static_cast<__half*>(out)[at] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(x);
}

// o / l; zero for a row that saw nothing, NaN where l is.
__device__ __forceinline__ float kv4_normalised(float o, float l) { return l == 0.f ? 0.f : o / l; }
__device__ __forceinline__ float kv4_lse(float m, float l, bool natural) {
  return l == 0.f ? -INFINITY : natural ? m + logf(l) : (m + log2f(l)) * kLn2;
}

// Four neighbouring outputs; their alignment is only that of the buffer.
__device__ __forceinline__ void kv4_store_out4(void* out, size_t at, int32_t type, const float (&o)[4], float l) {
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = kv4_normalised(o[e], l);
  if (type != 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (type == 1) {
        const __half2 y = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&y);
      } else {
        const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&y);
      }
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(w[0], w[1]);
  } else if (type == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) kv4_store_out(out, at + e, type, x[e]);
  }
}

// Index of (sequence b, row r, head) of a segment's column; false if unused.
__device__ __forceinline__ bool kv4_column(const Kv4AttendParams& p, uint32_t b, uint32_t seg, uint32_t c,
                                           uint32_t cols, size_t& index) {
  const uint32_t col = (seg % p.col_groups) * cols + c;
  if (col >= p.rows * p.group) return false;
  index = (size_t(b) * p.rows + col / p.group) * p.q_heads + (seg / p.col_groups) * p.group + col % p.group;
  return true;
}

// The positions of this thread's 16 tokens of the stage at token tb, or null
// where positions are indices (or the page is not there).
__device__ __forceinline__ const int32_t* kv4_positions(const Kv4AttendParams& p, uint32_t b, uint32_t h,
                                                        uint32_t len, uint32_t tb) {
  if (p.pool.pos == nullptr) return nullptr;
  const uint32_t t = tb + 16 * (threadIdx.x & 3);
  const uint32_t page = t < len ? kv4_load(p.table + size_t(b) * p.table_stride + (t >> p.log2_page)) : kNoUnit;
  if (page >= p.pool.pages) return nullptr;
  return p.pool.pos + (size_t(page) * p.pool.kv_heads + h) * p.page_tokens + (t & (p.page_tokens - 1));
}

__device__ __forceinline__ void kv4_report_lengths(const Kv4AttendParams& p) {
  if (blockIdx.x != 0) return;
  for (uint32_t b = threadIdx.x; b < p.batch; b += kKv4Threads)
    if (kv4_load(p.seq_lens + b) > p.max_tokens) atomicMax(&g_kvb_status, kKv4LenClamped);
}

template <int D, int C, int PD, int MINB, int RULES>
__global__ void __launch_bounds__(kKv4Threads, MINB) attend_kv4_kernel(const Kv4AttendParams p) {
  using S = Kv4Smem<D, true>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = lane >> 2, tig = lane & 3;
  Kv4Feeder<D, true, RULES> feed;
  feed.init(smem, warp);
  const uint32_t worker = blockIdx.x * kKv4Warps + warp;
  const uint32_t segs = p.pool.kv_heads * p.col_groups;
  Kv4Cursor cur;
  const uint32_t count = kv4_start<D, true, RULES>(p, worker, segs, C, cur);
  kv4_report_lengths(p);
  if (count == 0 && (!p.direct || worker >= p.workers)) return;

  feed.cur = cur;
  feed.next = 0;
  feed.count = count;
  feed.segs = segs;
  Kv4RawQuery<D> raw;
  feed.lookup(p);
  kv4_fetch_query<D, C>(p, cur.b, cur.seg / p.col_groups, cur.seg % p.col_groups, raw);
  if (count != 0) {
    feed.template copy<false>(p);
    feed.template copy<true>(p);
    feed.lookup(p);
  }
  uint32_t done = 0;
  const uint32_t vpitch = kv4_v_pitch(p.page_tokens * (D / 2), p.page_tokens);

  do {  // pieces
    const uint32_t first = done, end = min(count, uint32_t(cur.base + int32_t(cur.stages)));
    const uint32_t h = cur.seg / p.col_groups;
    Kv4Query<D, C> qf;
    kv4_make_query<D, C, RULES>(p, cur.b, h, cur.seg % p.col_groups, cur.len, raw, qf);
    const int32_t prefix = RULES && p.rule.prefix != nullptr ? int32_t(kv4_load(p.rule.prefix + cur.b)) : 0;
    Kv4State<D> st;
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[j][e] = 0.f;
    st.m = -INFINITY;
    st.l = st.lo = 0.f;
    for (; done < end; ++done) {
      const uint32_t j = uint32_t(int32_t(done) - cur.base);
      const uint32_t tb = (RULES && j >= cur.head ? j + cur.skip : j) * kStageTokens;
      const int32_t* pos = RULES == kRulesAll ? kv4_positions(p, cur.b, h, cur.len, tb) : nullptr;
      copy_wait<1>();  // K has landed, V may be on its way
      __syncwarp();
      float sc[kv4_tokens(C)];
      uint32_t digit[kv4_p_tiles(PD)][2][4], seen;
      float out_scale;
      kv4_dots<D, C>(feed.slots, qf, sc);
      const bool all = kv4_all_visible<RULES>(p, tb, cur.len, prefix);
      seen = kv4_scores<C, RULES>(p, feed.slots + S::kOffKp, tb, cur.len, prefix, all, qf.sum, qf.slope, qf.pos, pos, sc);
      copy_wait<0>();  // V has landed
      __syncwarp();    // and every lane has read K
      if (done + 1 < count) feed.template copy<false>(p);
      if (all)
        kv4_softmax<D, C, PD, RULES, false>(feed.slots + S::kOffVp, seen, sc, st, digit, out_scale);
      else
        kv4_softmax<D, C, PD, RULES, true>(feed.slots + S::kOffVp, seen, sc, st, digit, out_scale);
      kv4_output<D, PD>(feed.slots + S::kOffV, p.page_tokens, vpitch, digit, out_scale, st);
      __syncwarp();  // every lane has read V
      if (done + 1 < count) {
        feed.template copy<true>(p);
        feed.lookup(p);
      }
    }

    if (RULES && prefix < 0 && lane == 0) atomicMax(&g_kvb_status, kKv4LenClamped);
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 1);
    st.l += __shfl_xor_sync(0xffffffffu, st.l, 2);
    st.lo += __shfl_xor_sync(0xffffffffu, st.lo, 1);
    st.lo += __shfl_xor_sync(0xffffffffu, st.lo, 2);
    if (C == 4) {
      st.l += __shfl_xor_sync(0xffffffffu, st.l, 16);
      st.lo += __shfl_xor_sync(0xffffffffu, st.lo, 16);
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (C == 4) st.o[j][e] += __shfl_xor_sync(0xffffffffu, st.o[j][e], 16);
        st.o[j][e] += st.lo;
      }
    // The whole segment: the output; else a partial.
    const bool whole = int32_t(first) == cur.base && end - first == cur.stages;
    const uint32_t segment = cur.b * segs + cur.seg;
    size_t index;
    if (grp < C && kv4_column(p, cur.b, cur.seg, grp, C, index)) {
      if (whole) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) kv4_store_out4(p.out, index * D + 16 * j + 4 * tig, p.type, st.o[j], st.l);
        if (tig == 0 && p.lse != nullptr) p.lse[index] = kv4_lse(st.m, st.l, RULES == kRulesAll);
      } else {
        const size_t at = size_t(worker + segment) * C + grp;
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
          *reinterpret_cast<float4*>(p.part + at * D + 16 * j + 4 * tig) =
              make_float4(st.o[j][0], st.o[j][1], st.o[j][2], st.o[j][3]);
        if (tig == 0) p.part_ml[at] = make_float2(st.m, st.l);
      }
    }
    if (lane == 0 && !p.direct) {
      if (int32_t(first) == cur.base) p.seg_warps[segment].x = worker;
      if (int32_t(end) == cur.base + int32_t(cur.stages)) p.seg_warps[segment].y = worker;
    }
    if (done < count) {
      kv4_next_segment<RULES>(p, segs, cur);
      kv4_fetch_query<D, C>(p, cur.b, cur.seg / p.col_groups, cur.seg % p.col_groups, raw);
    }
  } while (done < count);
}

// The partials of one output row (sequence, row, head): out = sum o_i
// exp(m_i - m) / sum l_i exp(m_i - m). Bound by latency (3 to 4 us a call): two
// round trips, the segment's warps and then HELD of a row's partials a warp
// with their maxima and sums. Many partials a row: a CTA's 16 warps
// share a row, a thread per partial for the weights; few: a warp a row, a lane
// per partial.
constexpr int kKv4MergeWarps = 16;

template <int D>
struct Kv4Partial {
  static constexpr int kPer = D / 32;  // consecutive dims of a lane
  float x[kPer];
  __device__ __forceinline__ void load(const float* src) {
    const uint32_t lane = threadIdx.x & 31;
    if constexpr (D == 64) {
      const float2 y = __ldcg(reinterpret_cast<const float2*>(src) + lane);
      x[0] = y.x, x[1] = y.y;
    } else {
#pragma unroll
      for (int k = 0; k < D / 128; ++k) {
        const float4 y = __ldcg(reinterpret_cast<const float4*>(src) + lane * (D / 128) + k);
        x[4 * k] = y.x, x[4 * k + 1] = y.y, x[4 * k + 2] = y.z, x[4 * k + 3] = y.w;
      }
    }
  }
  __device__ __forceinline__ void add_to(float (&o)[kPer], float f) const {
#pragma unroll
    for (int k = 0; k < kPer; ++k) o[k] = fmaf(x[k], f, o[k]);
  }
};

// HELD: partials a warp has in flight at dim 128. Eight (64 registers a thread:
// a CTA can start beside the attention's last ones), or sixteen where a row has
// so many that eight would take another round.
template <int D, int RULES, bool MANY, int HELD>
__global__ void __launch_bounds__(32 * kKv4MergeWarps, HELD == 8 ? 2 : 1) merge_kv4_kernel(const Kv4AttendParams p, uint32_t cols) {
  __shared__ float sum[MANY ? kKv4MergeWarps : 1][MANY ? D : 1];
  __shared__ float weight[MANY ? 32 * kKv4MergeWarps : 1], part_max[kKv4MergeWarps], part_sum[kKv4MergeWarps];
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t index = MANY ? blockIdx.x : blockIdx.x * kKv4MergeWarps + warp;
  grid_launch_dependents();
  if (index >= p.batch * p.rows * p.q_heads) return;  // (few partials: warps do not meet)
  const uint32_t head = index % p.q_heads, br = index / p.q_heads;
  const uint32_t r = br % p.rows, b = br / p.rows, h = head / p.group;
  const uint32_t col = r * p.group + head % p.group, seg = h * p.col_groups + col / cols, c = col % cols;
  const uint32_t segment = b * p.pool.kv_heads * p.col_groups + seg;
  grid_dependency_wait();
  const uint2 range = __ldcg(p.seg_warps + segment);  // of a segment with stages
  const bool any = kv4_stage_count<RULES>(p, b) != 0;
  if (any && range.x == range.y) return;  // written by its warp
  const uint32_t n = any ? range.y - range.x + 1 : 0u;
  const size_t first = size_t(range.x + segment) * cols + c;
  constexpr int kPer = D / 32;
  constexpr int kHeld = D == 256 ? HELD / 2 : HELD;
  constexpr uint32_t kRound = MANY ? kHeld * kKv4MergeWarps : kHeld, kStep = MANY ? kKv4MergeWarps : 1;
  float o[kPer] = {}, top = -INFINITY, l = 0.f;
  for (uint32_t from = 0; from < n; from += kRound) {
    const uint32_t here = min(n - from, kRound), mine = MANY ? tid : lane, start = MANY ? warp : 0u;
    const float2 ml = mine < here ? __ldcg(p.part_ml + first + size_t(from + mine) * cols) : make_float2(-INFINITY, 0.f);
    Kv4Partial<D> held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (start + i * kStep < here) held[i].load(p.part + (first + size_t(from + start + i * kStep) * cols) * D);
    float m = warp_max(ml.x);
    if constexpr (MANY) {
      if (lane == 0) part_max[warp] = m;
      __syncthreads();
      m = warp_max(lane < kKv4MergeWarps ? part_max[lane] : -INFINITY);
    }
    m = fmaxf(m, top);
    const float sub = m == -INFINITY ? 0.f : m;
    const float f = kv4_exp<RULES>(ml.x, sub), alpha = kv4_exp<RULES>(top, sub);
    top = m;
    float s = warp_sum(ml.y * f);
    if constexpr (MANY) {
      weight[tid] = f;
      if (lane == 0) part_sum[warp] = s;
      __syncthreads();
      s = warp_sum(lane < kKv4MergeWarps ? part_sum[lane] : 0.f);
    }
    l = fmaf(l, alpha, s);
#pragma unroll
    for (int k = 0; k < kPer; ++k) o[k] *= alpha;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const float g = MANY ? weight[(start + i * kStep) % (32 * kKv4MergeWarps)] : __shfl_sync(0xffffffffu, f, i);
      if (start + i * kStep < here) held[i].add_to(o, g);
    }
    if constexpr (MANY) __syncthreads();  // the weights are read
  }
  if constexpr (MANY) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) sum[warp][lane * kPer + k] = o[k];
    __syncthreads();
    for (uint32_t d = tid; d < D; d += 32 * kKv4MergeWarps) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < kKv4MergeWarps; ++w) x += sum[w][d];
      kv4_store_out(p.out, size_t(index) * D + d, p.type, kv4_normalised(x, l));
    }
    if (tid != 0) return;
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      kv4_store_out(p.out, size_t(index) * D + lane * kPer + k, p.type, kv4_normalised(o[k], l));
    if (lane != 0) return;
  }
  if (p.lse != nullptr) p.lse[index] = kv4_lse(top, l, RULES == kRulesAll);
}

// ---------------------------------------------------------------------------
// Accumulated weights: the scores again, against the given log-sum-exp, for
// one group of query columns a launch. The segments are (sequence, KV head);
// one thread adds up a token's weight in a fixed order, so there are no
// atomics, and the groups' launches follow one another. (One launch over all
// groups needs every group's digits in registers, or atomics, whose order
// changes the sums.) Reads half of what attention does and a float a token,
// writes the float. Bound by the instructions of the scores: 32 sequences of
// 1K to 32K tokens, eight columns, take 82 us, 4.2 TB/s; 5,000 tokens 5.5 to 6.2
// us, a kernel's latency. K and the weights are read again for every eight
// columns: 16 x 4,096 tokens take 15 us with 8, 28 with 16, 80 with 48 and 208
// with 128.

template <int D, int C, int MINB, int RULES>
__global__ void __launch_bounds__(kKv4Threads, MINB) weigh_kv4_kernel(const Kv4AttendParams p, uint32_t group) {
  using S = Kv4Smem<D, false>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, grp = lane >> 2, tig = lane & 3;
  Kv4Feeder<D, false, RULES> feed;
  feed.init(smem, warp);
  const uint32_t segs = p.pool.kv_heads;  // p.col_groups is 1 here
  Kv4Cursor cur;
  const uint32_t count = kv4_start<D, false, RULES>(p, blockIdx.x * kKv4Warps + warp, segs, C, cur);
  kv4_report_lengths(p);
  if (count == 0) return;
  feed.cur = cur;
  feed.next = 0;
  feed.count = count;
  feed.segs = segs;
  feed.lookup(p);
  feed.template copy<false>(p);
  feed.lookup(p);
  uint32_t done = 0;

  while (done < count) {
    const uint32_t end = min(count, uint32_t(cur.base + int32_t(cur.stages)));
    Kv4RawQuery<D> raw;
    kv4_fetch_query<D, C>(p, cur.b, cur.seg, group, raw);
    Kv4Query<D, C> qf;
    kv4_make_query<D, C, RULES>(p, cur.b, cur.seg, group, cur.len, raw, qf);
    // Infinite: a column that is not there, or a row that saw nothing.
    float lse = INFINITY;
    const uint32_t col = group * C + grp % C;
    if (col < p.rows * p.group) {
      const float x = kv4_load(p.lse_in + (size_t(cur.b) * p.rows + col / p.group) * p.q_heads + cur.seg * p.group +
                            col % p.group);
      if (x != -INFINITY) lse = RULES == kRulesAll ? x : x * kLog2e;
    }
    const int32_t prefix = RULES && p.rule.prefix != nullptr ? int32_t(kv4_load(p.rule.prefix + cur.b)) : 0;
    float* weights = p.weights + (int64_t(cur.b) * p.pool.kv_heads + cur.seg) * p.weight_stride;
    for (; done < end; ++done) {
      const uint32_t j = uint32_t(int32_t(done) - cur.base);
      const uint32_t tb = (RULES && j >= cur.head ? j + cur.skip : j) * kStageTokens;
      const int32_t* pos = RULES == kRulesAll ? kv4_positions(p, cur.b, cur.seg, cur.len, tb) : nullptr;
      // After the reduction below this lane holds token t0 and the next.
      const uint32_t t0 = tb + 16 * tig + (C == 8 ? 2 * grp : 8 * (grp >> 1 & 1) + 4 * (grp >> 2) + 2 * (grp & 1));
      const float old0 = t0 < cur.len ? weights[t0] : 0.f, old1 = t0 + 1 < cur.len ? weights[t0 + 1] : 0.f;
      copy_wait<0>();
      __syncwarp();
      constexpr int kTokens = kv4_tokens(C);
      float w[kTokens];
      kv4_dots<D, C>(feed.slots, qf, w);
      uint32_t seen = kv4_scores<C, RULES>(p, feed.slots + S::kOffKp, tb, cur.len, prefix,
                                  kv4_all_visible<RULES>(p, tb, cur.len, prefix), qf.sum, qf.slope, qf.pos, pos, w);
      const bool absent = reinterpret_cast<const float*>(feed.slots + S::kOffKp + kv4_params_at<C>())[0] == kKv4Absent;
      __syncwarp();  // every lane has read K
      if (done + 1 < count) {
        feed.template copy<false>(p);
        feed.lookup(p);
      }
      if (lse == INFINITY || absent) seen = 0;
#pragma unroll
      for (int u = 0; u < kTokens; ++u) w[u] = seen >> u & 1u ? kv4_exp<RULES>(w[u], lse) : 0.f;
      // Sum over the columns (lanes grp % C), halving the tokens held at each
      // step; two are left: with 8 columns tokens 2 grp and the next, with 4
      // tokens 4 (grp / 4) + 8 (grp / 2 % 2) + 2 (grp % 2).
#pragma unroll
      for (int half = kTokens / 2; half >= 2; half >>= 1) {
        const uint32_t bit = 2 * half;
        const bool upper = lane & bit;
#pragma unroll
        for (int t = 0; t < half; ++t) {
          const float give = upper ? w[t] : w[t + half];
          const float keep = upper ? w[t + half] : w[t];
          w[t] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
        }
      }
      if (t0 < cur.len) weights[t0] = old0 + w[0];
      if (t0 + 1 < cur.len) weights[t0 + 1] = old1 + w[1];
    }
    if (RULES && prefix < 0 && lane == 0) atomicMax(&g_kvb_status, kKv4LenClamped);
    if (done < count) kv4_next_segment<RULES>(p, segs, cur);
  }
}

}  // namespace kvb
