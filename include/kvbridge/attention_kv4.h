#pragma once
// kvbridge-b200: a paged KV cache held in 4 bits, the attention that reads
// it, and its eviction by accumulated attention weight. Beside the int8 and
// fp32 caches of attention_common.h, which it leaves as they are.
//
// Row format. The `dim` values x of one token and KV head are held as codes
// 0..15 against the row's own range:
//   lo = min x, scale = (max x - min x) * (1.0f / 15.0f)      (all in fp32)
//   code = clamp(rint((x - lo) / scale), 0, 15)               (ties to even)
//   value = lo + scale * code
// A row of equal values has scale 0 and codes 0. A row that holds a value
// that is not finite (or whose range is not) has scale = lo = NaN and codes
// 0, so that attention that sees it returns NaN and attention that does not
// is untouched.
//
// Pool layout (dim 64, 128 or 256; page_tokens 16, 32 or 64), for page p, KV
// head h, slot s of the page, unit = p * kv_heads + h:
//   k         uint8[(unit * page_tokens + s) * dim / 2 + d / 2]
//   v         uint8[(unit * dim / 2 + d / 2) * page_tokens + s]
//             dim d in the low half of the byte for even d, the high half for odd d
//   k_params  float[(unit * page_tokens + s) * 2]   {scale, lo}
//   v_params  float[(unit * page_tokens + s) * 2]   {scale, lo}
//   positions int32[unit * page_tokens + s] or null: the token's position in
//             its sequence, not negative. Without it a token's position is
//             its index in the sequence's block table; a cache that has been
//             compacted needs it wherever positions matter (bias by distance,
//             window, prefix, several query rows).
// 2 * (dim / 2 + 8) bytes a token and KV head: 144 at dim 128, where the
// int8 layout takes 264.
//
// Arithmetic. Sums, softmax statistics, the log-sum-exp and the weights are
// fp32. Two values are held in fixed point: a query element to 2^-22 of its row's
// largest (in fp32 rows too), and the product of a probability and a V scale to
// 2^-16 (fp32 outputs 2^-23) of the largest of 64 tokens. Both stay far below
// what the 4-bit codes leave open, half a step of every value.
//
// Entry points throw std::invalid_argument before anything is enqueued for
// bad metadata or null or misaligned buffers, and std::runtime_error for
// CUDA failures. Every buffer is a device pointer that the caller owns; the
// library allocates nothing. Slots, page ids and lengths are read on the
// device: an invalid one is skipped (a length clamped) and reported through
// read_device_status (4 page id, 5 length, 6 slot, 8 kept token). No query row
// sees the tokens of a page id that is not in the pool, and their weights stay.
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

namespace kvbridge {

// Element types of dense rows, queries and outputs.
enum class Kv4Type : int32_t { f32 = 0, f16 = 1, bf16 = 2 };

struct Kv4Pool {
  uint32_t kv_heads, dim, page_tokens, pages;
  uint8_t* k;
  uint8_t* v;
  float* k_params;
  float* v_params;
  int32_t* positions;  // optional
};
const char* kv4_pool_error(const Kv4Pool&) noexcept;  // geometry; null when valid

// Dense K and V rows of `tokens` tokens: element (t, h, d) at
// k[t * k_stride + h * dim + d], likewise v (strides in elements, so that
// rows can be columns of a fused projection's output). Token t belongs to
// physical slot slots[t] = page * page_tokens + slot (negative: skipped).
struct Kv4Rows {
  uint32_t tokens;  // 0: nothing is launched
  Kv4Type type;
  void* k;
  void* v;
  int64_t k_stride, v_stride;
  const int64_t* slots;      // int64[tokens]
  const int32_t* positions;  // int32[tokens]; required by append_kv4 iff the pool has positions
};
// Quantises the rows and writes them to their slots. The slots of one call
// are distinct.
void append_kv4(const Kv4Pool&, const Kv4Rows&, cudaStream_t);
// The inverse: writes the values that the slots hold to the rows, rounded to
// the rows' type. Rows of skipped slots (negative or out of range) are zero.
void load_kv4(const Kv4Pool&, const Kv4Rows&, cudaStream_t);

// Queries: `rows` query rows of each of `batch` sequences, element
// (b, r, head, d) at q[b * batch_stride + r * row_stride + head * dim + d].
// Sequence b has seq_lens[b] cached tokens (its query rows' own K/V among
// them), at most max_tokens and at most table_stride * page_tokens; logical
// page j is physical page block_table[b * table_stride + j].
//
// Score of query row r (position pq) and token t (position pk):
//   x = scale * q . k
//   x = softcap * tanh(x / softcap)             if softcap > 0
//   x = x - slopes[head] * |pq - pk|            if slopes
// and t is visible iff t < seq_lens[b] and
//   (pk <= pq and (window == 0 or pq - pk < window)) or pk < prefix_lens[b].
// pq = q_positions[b * rows + r], or seq_lens[b] - rows + r without them.
struct Kv4Query {
  uint32_t batch, rows, q_heads, table_stride, max_tokens;
  Kv4Type type;  // of q and of the attention output
  float scale, softcap;
  uint32_t window;
  const void* q;
  int64_t batch_stride, row_stride;
  const uint32_t* seq_lens;     // uint32[batch]
  const uint32_t* block_table;  // uint32[batch * table_stride]
  const int32_t* q_positions;   // int32[batch * rows], optional; required iff the pool has positions
  const float* slopes;          // float[q_heads], optional
  const uint32_t* prefix_lens;  // uint32[batch], optional; 2^31 and more: 0, and reported as a length
};
const char* kv4_query_error(const Kv4Pool&, const Kv4Query&) noexcept;

// Bytes of 16-byte aligned workspace that launch_attention_kv4 needs on the
// current device.
size_t attention_kv4_workspace_bytes(const Kv4Pool&, const Kv4Query&);
// out (the query's type, [batch][rows][q_heads][dim]) = sum softmax(x) v;
// lse (float[batch * rows * q_heads], optional) = ln sum exp(x). A query row
// that sees no token gets zeros and -inf.
void launch_attention_kv4(const Kv4Pool&, const Kv4Query&, void* workspace, size_t workspace_bytes,
                          void* out, float* lse, cudaStream_t);

// weights[(b * kv_heads + h) * weight_stride + t] += the attention weight
// that token t of sequence b got in this step from the query rows and the
// query heads of KV head h: sum of exp(x - lse) where visible, with the lse
// of launch_attention_kv4. Weights belong to a sequence, not to a page, so
// sequences may share pages. Fixed order of summation.
void accumulate_weights_kv4(const Kv4Pool&, const Kv4Query&, const float* lse, float* weights,
                            int64_t weight_stride, cudaStream_t);

// Eviction. Of the seq_lens[b] tokens of sequence b and KV head h the first
// `sinks`, the last `recent` and, among the rest, those of the largest
// accumulated weight are kept, `budget` in all (ties keep the lower index, a
// NaN weight counts as the largest). A sequence of at most `budget` tokens
// keeps them all.
struct Kv4Eviction {
  uint32_t batch, kv_heads, max_tokens, budget, sinks, recent;
  const uint32_t* seq_lens;  // uint32[batch], each <= max_tokens
  const float* weights;      // element (b, h, t) at (b * kv_heads + h) * weight_stride + t
  int64_t weight_stride;     // at least max_tokens
};
const char* kv4_eviction_error(const Kv4Eviction&) noexcept;
// keep: int32[batch * kv_heads * budget], the kept tokens of each (b, h) in
// ascending order, then zeros; kept_lens: uint32[batch] = min(seq_lens[b],
// budget), not in the place of seq_lens. Works for any cache that keeps weights.
void select_tokens(const Kv4Eviction&, int32_t* keep, uint32_t* kept_lens, cudaStream_t);
// Copies the kept tokens (codes, parameters, positions) of every sequence
// and KV head in order to the pages new_table[b * new_stride + j] of the
// same pool, which no block table of the call may use, and their weights to
// new_weights (optional; `budget` values a row, zeros after the kept ones,
// rows new_weight_stride apart, none in the place of the old ones). A kept
// token beyond its sequence, beyond the block table's row or on a page that is
// not in the pool is reported, and its new slot holds a row of NaN (position
// 0). The old pages are only read, so sequences may share them; the caller
// frees them afterwards.
void compact_kv4(const Kv4Pool&, const Kv4Eviction&, const uint32_t* block_table,
                 uint32_t table_stride, const int32_t* keep, const uint32_t* new_table,
                 uint32_t new_stride, float* new_weights, int64_t new_weight_stride, cudaStream_t);

namespace detail {
// Status word of the kernels of this header (they live in their own module and
// wait for nothing but the kernel before); read_device_status includes it.
cudaError_t read_kv4_status(int* status) noexcept;
}  // namespace detail

}  // namespace kvbridge
