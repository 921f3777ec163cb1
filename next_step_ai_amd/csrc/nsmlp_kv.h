// Paged K/V cache in 8 or 4 bits: layouts, argument blocks and device helpers
// shared by the bookkeeping kernels (nsmlp_kv.hip), those of the 4-bit format
// and the rotation (nsmlp_kv4.hip) and the attention (nsmlp_attention.hip).
//
// Layout in 8 bits.  A block holds B tokens (16, 32 or 64) of every K/V head.  Its bytes
// are [kv_heads][2: K, V][B * D]; a (block, head)'s K and V are runs of B/16
// tiles of 16 tokens, 16 D bytes each, ordered so that 64 lanes reading 16
// bytes each at consecutive addresses hold an MFMA operand:
//   K tile  [D/16][16 tokens][16 dims]
//   V tile  [D/64][4 token groups][64 dims][4 tokens]
// One 16x16x32 product of K (rows: tokens) with queries (columns) leaves token
// 4 g + i of a query in lane group g = lane / 16, register i; that is where
// the product of V (rows: dims) with the weights wants them, so weights need
// no exchange between lanes.
// scale [blocks][kv_heads][2] fp32: value = code * scale.
//
// Layout in 4 bits (NSMLP_KV_E2M1).  A (block, head) is a run of K codes, V
// codes, K scales and V scales, each a run of B/16 tiles of 16 tokens.  A code
// is an e2m1 nibble, a byte two neighbouring dims of a token (the lower dim in
// the low nibble), a scale byte a power of two, 2^(byte - 127), of 32 dims of a
// token.  With r = 16th part of the dims (D/16 of them) and w = D/32 bytes:
//   K tile  [4 quarters of the dims][16 tokens][D/4 dims]           8 D bytes
//   V tile  [4 token groups][16 r][4 tokens][D/16 dims]             8 D bytes
//   K scale [D/32][16 tokens], V scale [4 token groups][D/32][4 tokens]
// so that a lane's 16 (or 8) bytes are its operand of the same products: K's
// under one scale, V's 4 tokens under one scale each, which a conversion to fp16
// applies on the way.  A token's bytes are its own in both, so that tokens are
// stored without reading what stands next to them.
#pragma once

#include "nsmlp_internal.h"

namespace nsmlp {

constexpr int kKvTile = 16;
constexpr float kKvScaleMin = 7.888609052210118e-31f;  // 2^-100

struct KvView {
  uint8_t* data;
  float* scale;
  int num_blocks, heads, D, B, b_shift, fmt;  // fmt: NSMLP_KV_INT8 / NSMLP_KV_E4M3 / NSMLP_KV_E2M1
};

// bytes of a (block, head), K and V
template <int kFmt>
__host__ __device__ constexpr int kv_block_bytes(int B, int D) {
  return kFmt == NSMLP_KV_E2M1 ? B * D + B * D / 16 : 2 * B * D;
}

// byte of (token t, dim d) inside a (block, head)'s K or V
__host__ __device__ __forceinline__ int kv_k_off(int D, int t, int d) {
  return (t >> 4) * 16 * D + (d >> 4) * 256 + (t & 15) * 16 + (d & 15);
}
__host__ __device__ __forceinline__ int kv_v_off(int D, int t, int d) {
  return (t >> 4) * 16 * D + (d >> 6) * 1024 + ((t & 15) >> 2) * 256 + (d & 63) * 4 + (t & 3);
}

// The same of the 4-bit format: where the D/16 dims from D/16 * r of token t
// start in K and in V (codes), and the byte of its 32 dims' scale.
__host__ __device__ __forceinline__ int kv4_k_off(int D, int t, int r) {
  return (t >> 4) * 8 * D + ((r >> 2) * 16 + (t & 15)) * (D / 8) + (r & 3) * (D / 32);
}
__host__ __device__ __forceinline__ int kv4_v_off(int D, int t, int r) {
  return (t >> 4) * 8 * D + (((t & 15) >> 2) * 16 + r) * (D / 8) + (t & 3) * (D / 32);
}
__host__ __device__ __forceinline__ int kv4_ks_off(int D, int t, int group) { return (t >> 4) * (D / 2) + group * 16 + (t & 15); }
__host__ __device__ __forceinline__ int kv4_vs_off(int D, int t, int group) {
  return (t >> 4) * (D / 2) + (((t & 15) >> 2) * (D / 32) + group) * 4 + (t & 3);
}
// The scales' exponents: a code times 2^-23 to 2^13 is an fp16 number, subnormal
// ones among them.  255 in K's scales marks a token whose K or V is not finite.
constexpr int kKv4Least = -23, kKv4Most = 13;
constexpr uint32_t kKv4Bad = 255;

// int8 codes are stored with 128 added, so that a byte next to 0x64 is the
// fp16 value 1024 + 128 + code: two permutes and two packed subtractions turn
// a dword into four exact fp16 codes.  e4m3 codes are stored as they are.
template <int kFmt>
__device__ __forceinline__ float kv_decode1(uint32_t byte) {
  if constexpr (kFmt == NSMLP_KV_INT8) return (float)((int)byte - 128);
  else return __builtin_amdgcn_cvt_f32_fp8(byte, 0);
}

// four codes of a dword as fp16, in byte order
template <int kFmt>
__device__ __forceinline__ uint2 kv_half4(uint32_t w) {
  if constexpr (kFmt == NSMLP_KV_INT8) {
    const half2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    const half2_t lo = as_half2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias;
    const half2_t hi = as_half2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias;
    return uint2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  } else {
    const half2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    const half2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    return uint2{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
  }
}

// The scale that a largest magnitude asks for.  int8: a times fp32(1 / 127).  e4m3: the
// smallest power of two that keeps a within 448, so that recoding a block
// under a larger scale moves exponents and rounds subnormals only.  Never
// below 2^-100; NaN where a is not finite.
template <int kFmt>
__device__ __forceinline__ float kv_scale_of(float a) {
  if (!(a < INFINITY)) return __uint_as_float(0x7FC00000u);
  float s;
  if constexpr (kFmt == NSMLP_KV_INT8) {
    s = a * (1.0f / 127.0f);
  } else {
    int e = 0;
    const float m = frexpf(a, &e);  // a = m 2^e, m in [0.5, 1)
    s = a == 0.0f ? 0.0f : ldexpf(1.0f, m <= 0.875f ? e - 9 : e - 8);
  }
  return fmaxf(s, kKvScaleMin);
}

// Angles by position, and the query rows that an append rotates on the way.
struct KvRotateArgs {
  const float* table;        // [reach][D / 2][2] cos, sin; NULL: no rotation
  const int32_t* positions;  // [n]
  int reach, interleaved;
  const uint16_t* q;  // [n][q_heads][D] or NULL
  uint16_t* q_out;
  long long q_row, q_head, out_row, out_head;  // strides in elements
  int q_heads;
  unsigned first;  // workgroup of the first query rows (set by the launch)
};

struct KvAppendArgs {
  KvView c;
  const uint16_t *k, *v;
  long long k_row, k_head, v_row, v_head;  // strides in elements
  const int64_t* slots;
  int n;
  int take;  // tokens that a wave looks at (set by the launch)
  KvRotateArgs rot;
};
void launch_kv_append(const KvAppendArgs& a, bool bf16, hipStream_t s);   // 8 bits
void launch_kv_append4(const KvAppendArgs& a, bool bf16, hipStream_t s);  // 4 bits

struct KvReadArgs {
  KvView c;
  const int64_t* slots;
  int n;
  uint16_t *k, *v;  // [n][heads][D]
};
void launch_kv_read(const KvReadArgs& a, bool bf16, hipStream_t s);
void launch_kv_read4(const KvReadArgs& a, bool bf16, hipStream_t s);

// Work of an attention call, listed by the step's plan.  A unit is up to
// `rows` query rows of a request (row = token * group + head of the group)
// against keys [kv_begin, kv_end) of every K/V head.  Two lists:
//   a  requests whose rows fit one tile of 16 (or any that a step without list b
//      refuses for their length): their keys are streamed.  All
//      these requests' keys, one after the other in pieces of 64, are cut into
//      equal shares, one per workgroup and K/V head; a unit is what a share
//      holds of a request.  A request's units meet in the last to end.
//   b  the others, in tiles of `rows_b` rows.  Where there are few tiles, a
//      tile's keys are cut into parts, which a second launch joins, one KvSplit
//      per tile.
struct KvUnit {
  int32_t req, row, kv_begin, kv_end;
  int32_t part, first, parts, pad;  // this unit's partial (-1: none); list a: the first of its rows', how many
};
struct KvSplit {
  int32_t req, row, first, parts;
};

constexpr int kKvMaxRequests = 4096;
constexpr int kKvRowsA = 16;
// arrival counters of a level of list a's joins, one per (partial, K/V head):
// at most 2 shares, and shares times heads is below 512 + heads (<= 1024); 4
// levels of 8 join 4096 parts, and there are at most 512
constexpr int kKvCounters = 8192;
static_assert(4 * kKvCounters <= kMaxK && 2 * (512 + 1024) <= kKvCounters, "the workspace's block counters");
constexpr int kKvHeaderInts = 16;  // units a, shares, units b, splits b

struct KvSchedule {  // sizes, from the host's knowledge of a step (kv_schedule)
  int rows_b, join_rows;             // rows of a tile of list b, and how many of them a request can fill
  int shares;                        // of list a's keys, at most
  int target_b;                      // CUs per K/V head that list b's keys are shared out to (0: they are not)
  int max_units_a, max_units_b;      // list capacities
  int max_parts_a, max_parts_b, max_splits_b;
  bool list_b;                       // whether a request can be long enough for list b
  long long off_shares, off_units_a, off_units_b, off_splits_b, ints;  // in ints
};
KvSchedule kv_schedule(int requests, int total, int max_new, int group, int kv_heads);

struct KvPlanArgs {
  int R, total, max_new, row_limit, max_blocks, num_blocks, B, b_shift, group;
  const int32_t *cached, *fresh;     // [R]
  int32_t* table;                    // [R][max_blocks]
  const int32_t *ring, *state;       // [num_blocks] free blocks, (head, count)
  int64_t* slots;                    // [total]
  int32_t* positions;                // [total] or NULL
  int32_t *q_start, *kv_len, *next;  // [R + 1], [R], [R]
  int32_t* info;                     // [4] head, count, refused, tokens
  int32_t* sched;
  KvSchedule s;
};
void launch_kv_plan(const KvPlanArgs& a, hipStream_t s);

struct KvAttnArgs {
  KvView c;
  const uint16_t* q;
  long long q_row, q_head;  // strides in elements
  uint16_t* out;            // [tokens][q_heads][D]
  float* lse;               // [tokens][q_heads] or NULL
  const int32_t *table, *q_start, *kv_len, *sched;
  int max_blocks, R, total, group;
  float scale_log2;  // softmax scale times log2(e)
  float *acc_a, *ml_a, *acc_b, *ml_b;  // partial results of either list: [parts][kv_heads][rows][D], [..][2] (m, l), [..][4] (m, l, x)
  int *status, *count;  // status word, arrival counters [levels][kKvCounters] (zero, left zero)
  KvSchedule s;
};
// floats of the partial results, and where acc_a, ml_a, acc_b, ml_b start
size_t kv_attn_partial_floats(const KvSchedule& s, int kv_heads, int D, size_t (&off)[4]);
void launch_kv_attention(const KvAttnArgs& a, bool bf16, hipStream_t s);

struct KvCommitArgs {
  int R, max_blocks, num_blocks, b_shift, B;
  int32_t *cached, *table, *ring, *state;
  const int32_t *next, *info;
  const int32_t* finished;  // [R] or NULL
};
void launch_kv_commit(const KvCommitArgs& a, hipStream_t s);

// f<D, format, bf16>(args) for the cache's head size and 8-bit format
#define NSMLP_KV_BY_TYPE(f, a, bf16, s)                                                            \
  do {                                                                                             \
    const bool i8_ = (a).c.fmt == NSMLP_KV_INT8;                                                   \
    if ((a).c.D == 128) {                                                                          \
      if (i8_) (bf16) ? f<128, NSMLP_KV_INT8, true>(a, s) : f<128, NSMLP_KV_INT8, false>(a, s);    \
      else (bf16) ? f<128, NSMLP_KV_E4M3, true>(a, s) : f<128, NSMLP_KV_E4M3, false>(a, s);        \
    } else {                                                                                       \
      if (i8_) (bf16) ? f<64, NSMLP_KV_INT8, true>(a, s) : f<64, NSMLP_KV_INT8, false>(a, s);      \
      else (bf16) ? f<64, NSMLP_KV_E4M3, true>(a, s) : f<64, NSMLP_KV_E4M3, false>(a, s);          \
    }                                                                                              \
  } while (0)

}  // namespace nsmlp
