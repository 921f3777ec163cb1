// Log probabilities of given tokens, entropies and the most likely tokens from
// the logits, in one pass over them.
//
// With m the largest logit of a row (finite), l = sum e^(z - m) and x = sum e^(z - m) (z - m):
//   log p_t = (z_t - m) - log l          entropy = log l - x / l
// Neither subtracts large numbers from each other, as z - log sum e^z would.  What
// the largest logit itself adds to l, 1, is kept apart, so that where one token has
// nearly all of a row log l = log(1 + r) is known to its own size (a log probability
// of -0.005 to 2e-7 of it; with the 1 in the sum to 1e-5).
// A wave's lanes have their sums (fp32) under one m, raised at most once per batch of
// vectors; waves and workgroups join theirs under the largest m.  A NaN or +inf makes
// l NaN; -inf adds nothing to l, and to x neither, as the factor z - m is held above
// -200, below which e^(z - m) is zero.
//
// The top n of a row are found as whole numbers (order of the logit, then the
// lower index first): 64 bits, all different.  A wave keeps the candidates above
// its n-th largest so far in LDS and drops all but n where they pass 2 n or 64; the first
// bound is the n-th largest of the lanes' own maxima of the first batch.  So nearly
// all vectors cost one comparison.  A NaN counts as below every number.
//
// What bounds it: many rows, the vector instructions, an exp2 and nine others for a
// logit, which are issued in 94% of the cycles: 2048 rows of 128256 in bf16 with 5
// alternatives (525 MB) 113 to 116 us, 4.6 TB/s, without alternatives 101, where a kernel
// that only reads takes 84 (6.25 TB/s).  In fp32, twice the bytes, 192 us (5.5 TB/s; in
// 75%).  One row, the chain of a load, the selection and the joins: 128256 in fp16 5.4 us
// without alternatives, 10.2 with 5, 26 with 64, where candidates are counted against
// each other.
//
// The sums are joined in the order of their workgroups, whoever ends last.  How many
// workgroups a row has depends on the number of rows, and with it the order of the
// fp32 sums: a row's numbers may differ in their last bits between calls of other rows.
#include <algorithm>
#include <type_traits>

#include "nsmlp_internal.h"

namespace nsmlp {

namespace {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / kWave;
constexpr int kLpBatch = 4;          // vectors of 16 bytes that a lane has in flight
constexpr int kLpMaxTop = 64;
constexpr int kLpMaxSplits = 32;
constexpr float kLog2e = 1.4426950408889634f, kLowest = -3.402823466e38f;

struct LogprobArgs {
  const uint8_t* logits;
  long long row_bytes;
  int rows, vocab, top, splits;
  int each;                // wave steps of a workgroup
  uint32_t per_split;      // ceil(2^20 / splits): k / splits of k < 2^11 + 2^8 as a product
  const int64_t* tokens;   // [rows] or NULL
  float *logprob, *entropy;  // [rows], nullable
  int64_t* top_ids;        // [rows][top]
  float* top_logprobs;
  float* part_sums;        // [rows][splits][4]: m, l, x, ones
  uint64_t* part_top;      // [rows][splits][top]
  int* count;              // [rows] workgroups of a row that have ended (zero, left zero)
};

enum class Logit { kF16, kBf16, kF32 };
template <Logit T>
constexpr int kPerVector = T == Logit::kF32 ? 4 : 8;

template <Logit T>
__device__ __forceinline__ float value_at(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (T == Logit::kF32) return __uint_as_float(w[i]);
  else if constexpr (T == Logit::kBf16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
  else return h2f((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
}
// the same for an index that is not known when compiled
template <Logit T>
__device__ __forceinline__ float value_of(const uint4& v, int i) {
  const int word = T == Logit::kF32 ? i : i >> 1;
  const uint64_t low = (uint64_t)v.y << 32 | v.x, high = (uint64_t)v.w << 32 | v.z;
  const uint32_t w = (uint32_t)((word & 2 ? high : low) >> (32 * (word & 1)));
  if constexpr (T == Logit::kF32) return __uint_as_float(w);
  else if constexpr (T == Logit::kBf16) return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  else return h2f((uint16_t)(w >> (16 * (i & 1))));
}
template <Logit T>
__device__ __forceinline__ float load_one(const uint8_t* row, long long i) {
  if constexpr (T == Logit::kF32) return reinterpret_cast<const float*>(row)[i];
  else if constexpr (T == Logit::kBf16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(row)[i] << 16);
  else return h2f(reinterpret_cast<const uint16_t*>(row)[i]);
}

// 16 bytes of a row from logit i on, at any address.
__device__ __forceinline__ uint4 vector_at(const uint8_t* p) {
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// A row of fewer logits than a vector has places: in its last ones.
template <Logit T>
__device__ __forceinline__ uint4 short_row(const uint8_t* row, int vocab) {
  constexpr int kPer = kPerVector<T>;
  uint32_t w[4] = {};
#pragma unroll
  for (int j = 1; j < kPer; ++j) {
    const int i = j - (kPer - vocab);
    if (i < 0) continue;
    if constexpr (T == Logit::kF32) w[j] = reinterpret_cast<const uint32_t*>(row)[i];
    else w[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[i] << (16 * (j & 1));
  }
  return uint4{w[0], w[1], w[2], w[3]};
}
// -inf in a vector's first `lost` places
template <Logit T>
__device__ __forceinline__ uint4 without(const uint4& v, int lost) {
  constexpr uint32_t kNone = T == Logit::kF32 ? 0xFF800000u : T == Logit::kBf16 ? 0xFF80FF80u : 0xFC00FC00u;
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (T == Logit::kF32) {
      w[j] = j < lost ? kNone : w[j];
    } else {
      const uint32_t gone = 2 * j + 1 < lost ? ~0u : 2 * j < lost ? 0xFFFFu : 0u;
      w[j] = (w[j] & ~gone) | (kNone & gone);
    }
  }
  return uint4{w[0], w[1], w[2], w[3]};
}

// A logit's place in the order: larger for a larger one, -0 as +0, 0 for NaN.
__device__ __forceinline__ uint32_t order_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.0f);
  return z != z ? 0u : (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
  return order == 0 ? __uint_as_float(0x7FC00000u) : __uint_as_float((int)order < 0 ? order & 0x7FFFFFFFu : ~order);
}
__device__ __forceinline__ uint64_t entry_of(float z, uint32_t index) { return (uint64_t)order_of(z) << 32 | (0xFFFFFFFFu - index); }
__device__ __forceinline__ uint32_t index_of(uint64_t entry) { return 0xFFFFFFFFu - (uint32_t)entry; }

// LDS writes of a wave are read by its other lanes: LDS keeps a wave's
// operations in order, this keeps the compiler's.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Largest of, and sum over, a wave's lanes: within rows of 16 through DPP, the four
// rows' through scalar registers (exchanges through LDS took most of the joins).
template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kCtrl, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_of(float v, int row) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16 * row)); }
__device__ __forceinline__ float wave_most(float v) {
  v = fmaxf(v, dpp<0x128>(v)), v = fmaxf(v, dpp<0x124>(v)), v = fmaxf(v, dpp<0x122>(v)), v = fmaxf(v, dpp<0x121>(v));  // row_ror
  return fmaxf(fmaxf(row_of(v, 0), row_of(v, 1)), fmaxf(row_of(v, 2), row_of(v, 3)));
}
__device__ __forceinline__ float wave_total(float v) {
  v += dpp<0x128>(v), v += dpp<0x124>(v), v += dpp<0x122>(v), v += dpp<0x121>(v);
  return (row_of(v, 0) + row_of(v, 1)) + (row_of(v, 2) + row_of(v, 3));
}

// How many of the entries in LDS (a multiple of 8, 16-byte aligned, 0 for none) are
// larger than each of `mine`.
template <int N>
__device__ __forceinline__ void count_above(const uint64_t* list, int count, const uint64_t (&mine)[N], int (&above)[N]) {
  const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(list);
#pragma unroll 1
  for (int j = 0; j < count; j += 8) {  // (eight are read at a time: one by one, each read was waited for)
    ulonglong2 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pairs[(j >> 1) + i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) above[k] += (v[i].x > mine[k]) + (v[i].y > mine[k]);
  }
}

// Candidates of a wave: entries in LDS, of which the n largest count.  They are
// settled where they pass `limit`: late enough for as many as n new ones (with a
// limit of 64 candidates, 64 alternatives of 1200 rows of 50257 took 117 us, so 82;
// one row of 128256 32, so 25), and no later, as the bound rises then.
constexpr int kLpList = 3 * kWave;
struct WaveTop {
  uint64_t* buf;          // [kLpList]
  int n, count, limit;    // (the same in all lanes)
  uint64_t bound;  // entries at or below it are not among the n largest
  float least;     // what a logit of the next batch has to reach (-inf: any may count)
  int lane;

  __device__ __forceinline__ void start(uint64_t* b, int top, int l) {
    buf = b, n = top, count = 0, limit = max(kWave, 2 * n), bound = 0, least = -INFINITY, lane = l;
  }

  // The n largest, in order, and the bound that follows.  An entry's place is the
  // number of larger ones; 0 stands for none.
  template <int N>
  __device__ __forceinline__ void rank() {
    uint64_t mine[N];
    int above[N] = {};
#pragma unroll
    for (int k = 0; k < N; ++k) mine[k] = buf[lane + k * kWave];
    count_above<N>(buf, count, mine, above);
    wave_sync();
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (lane + k * kWave < count && above[k] < n) buf[above[k]] = mine[k];
  }
  __device__ __forceinline__ void settle() {
    wave_sync();
    if (lane < 8 && count + lane < kLpList) buf[count + lane] = 0;
    wave_sync();
    if (count > 2 * kWave) rank<3>();
    else if (count > kWave) rank<2>();
    else rank<1>();
    wave_sync();
    if (count >= n) {
      count = n;
      bound = buf[n - 1];
      // a logit of a later batch stands behind its equals: the next larger one is the least that counts
      const uint32_t order = (uint32_t)(bound >> 32);
      least = least_of(order >= 0x007FFFFFu && order < 0xFF800000u ? order + 1 : order);
    }
  }
  // the logit of a place in the order, -inf for those of -inf and NaN
  static __device__ __forceinline__ float least_of(uint32_t order) { return order < 0x00800000u ? -INFINITY : logit_of(order); }
  // A first bound from the lanes' largest logits: what at least n of them reach.
  __device__ __forceinline__ void expect(float most) {
    uint32_t* orders = reinterpret_cast<uint32_t*>(buf);
    const uint32_t order = order_of(most);
    orders[lane] = order;
    wave_sync();
    const uint4* fours = reinterpret_cast<const uint4*>(orders);
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < kWave / 4; ++j) {
      const uint4 v = fours[j];
      above += (v.x > order) + (v.y > order) + (v.z > order) + (v.w > order);
    }
    wave_sync();
    // (the least of those with fewer than n above them)
    least = -wave_most(above < n ? -least_of(order) : kLowest);
  }
  // Every lane may bring an entry.
  __device__ __forceinline__ void offer(bool mine, uint64_t entry) {
    const bool in = mine && entry > bound;
    const unsigned long long who = __ballot(in);
    if (who == 0) return;
    if (in) buf[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = entry;
    count += __popcll(who);
    if (count > limit) settle();
  }
};

// Sums under a largest logit m: of the weights that are in `ones` (logits equal to m,
// some or all) and of the others.
struct Sums {
  float m, l, x, ones;
  __device__ __forceinline__ float all() const { return l + ones; }
};
__device__ __forceinline__ void rebase(Sums& s, float m) {
  const float d = s.m - m;
  if (d != 0.0f) {  // (NaN where both are inf)
    const float f = __builtin_amdgcn_exp2f(d * kLog2e), l = s.all();
    s.x = f * __builtin_fmaf(fmaxf(d, -200.0f), l, s.x);
    s.l = f * l;
    s.ones = 0.0f;
  }
  s.m = m;
}
__device__ __forceinline__ Sums join_lanes(const Sums& s) {  // of one m
  return Sums{s.m, wave_total(s.l), wave_total(s.x), wave_total(s.ones)};
}

__device__ __forceinline__ float log_prob(float z, const Sums& s, float log_l) {
  return s.all() == 0.0f ? -INFINITY : (z - s.m) - log_l;  // (nothing but -inf in the row)
}

// The row's results from its sums and, in `list`, its n largest.
template <Logit T>
__device__ __forceinline__ void write_row(const LogprobArgs& a, int row, const uint8_t* logits, const Sums& s, const uint64_t* list,
                                          int tid) {
  // the weights were 2^(d kLog2e) = e^(d (1 + kOff)), so that l is off by kOff x
  constexpr float kOff = -1.3349758e-8f;  // kLog2e as rounded, over log2 e, less 1
  const float l = s.all(), others = l == 0.0f ? 0.0f : __builtin_fmaf(-kOff, s.x, s.l);
  const float log_l = s.ones == 1.0f ? log1pf(others) : logf(others + s.ones);
  if (tid == 0) {
    if (a.logprob != nullptr) {
      const int64_t t = a.tokens[row];
      a.logprob[row] = t >= 0 && t < a.vocab ? log_prob(load_one<T>(logits, t), s, log_l) : __uint_as_float(0x7FC00000u);
    }
    if (a.entropy != nullptr) a.entropy[row] = l == 0.0f ? 0.0f : log_l - s.x / l;
  }
  if (tid < a.top) {
    const uint64_t e = list[tid];
    a.top_ids[(long long)row * a.top + tid] = (int64_t)index_of(e);
    a.top_logprobs[(long long)row * a.top + tid] = log_prob(logit_of((uint32_t)(e >> 32)), s, log_l);
  }
}

template <Logit T, bool kTop, bool kShort>
__global__ void __launch_bounds__(kLpThreads, 5) k_token_logprobs(LogprobArgs a) {
  kernarg_warm<sizeof(LogprobArgs)>();
  constexpr int kPer = kPerVector<T>, kSize = T == Logit::kF32 ? 4 : 2;
  __shared__ __attribute__((aligned(16))) uint64_t bufs[kLpWaves][kLpList];
  __shared__ uint64_t merged[kLpMaxTop];
  __shared__ float sums[kLpWaves][4];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = blockIdx.x, split = blockIdx.y;
  const uint8_t* logits = a.logits + (long long)row * a.row_bytes;
  const int steps = (a.vocab + kPer * kWave - 1) / (kPer * kWave);  // of a wave: 64 vectors
  const int first = split * a.each, end = min(first + a.each, steps);

  WaveTop top;
  if constexpr (kTop) top.start(bufs[wave], a.top, lane);
  Sums s = {kLowest, 0.0f, 0.0f, 0.0f};
  int ones = 0;  // of the wave
  for (int at = first + wave; at < end; at += kLpWaves * kLpBatch) {
    uint4 raw[kLpBatch];
    if constexpr (!kShort) {
#pragma unroll
      for (int u = 0; u < kLpBatch; ++u) {
        // one that would end past the row ends with it
        const long long i0 = ((long long)(at + u * kLpWaves) * kWave + lane) * kPer;
        raw[u] = vector_at(logits + min(i0, (long long)a.vocab - kPer) * kSize);
      }
    } else {
      raw[0] = short_row<T>(logits, a.vocab);
#pragma unroll
      for (int u = 1; u < kLpBatch; ++u) raw[u] = raw[0];
    }
    if (at + (kLpBatch - 1) * kLpWaves >= min(steps - 1, end)) {
      // -inf where there is no logit, or one that an earlier vector has
#pragma unroll
      for (int u = 0; u < kLpBatch; ++u) {
        const int step = at + u * kLpWaves;
        const long long i0 = ((long long)step * kWave + lane) * kPer;
        const int lost = step < end ? (int)min(max(i0 + kPer - a.vocab, 0LL), (long long)kPer) : kPer;
        raw[u] = without<T>(raw[u], lost);
      }
    }
    float most[kLpBatch];  // of a vector (NaN only where every one is)
#pragma unroll
    for (int u = 0; u < kLpBatch; ++u) {
      most[u] = value_at<T>(raw[u], 0);
#pragma unroll
      for (int j = 1; j < kPer; ++j) most[u] = fmaxf(most[u], value_at<T>(raw[u], j));
    }
    const float all = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    if (__ballot(all > s.m) != 0) {
      s.ones = lane == 0 ? (float)ones : 0.0f;
      rebase(s, wave_most(all));
      ones = 0;
    }
    const auto add = [&](auto has_most, int u) {
      float l = 0.0f, x = 0.0f;  // (a vector's sums first: fewer roundings on the way of each weight)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float d = value_at<T>(raw[u], j) - s.m, p = __builtin_amdgcn_exp2f(d * kLog2e);
        if constexpr (decltype(has_most)::value) {
          ones += __popcll(__ballot(d == 0.0f));
          l += d == 0.0f ? 0.0f : p;
        } else {
          l += p;
        }
        x = __builtin_fmaf(p, fmaxf(d, -200.0f), x);
      }
      s.l += l, s.x += x;
    };
    // Few batches of a long row hold an m (1 + log n of n, as a wave has one): those that
    // do not have no branch between their vectors.  (700 rows of 128256 with 5
    // alternatives 51.7 us, with a branch per vector in all batches 52.3, every vector of
    // a batch that raises m counted 53.7, with the 1 in the sum 48.5.)
    if (__builtin_expect_with_probability(__ballot(all == s.m) != 0, 0, 0.9)) {
#pragma unroll
      for (int u = 0; u < kLpBatch; ++u) {
        if (__ballot(most[u] == s.m) != 0) add(std::true_type{}, u);
        else add(std::false_type{}, u);
      }
    } else {
#pragma unroll
      for (int u = 0; u < kLpBatch; ++u) add(std::false_type{}, u);
    }
    if constexpr (kTop) {
      if (at == first + wave) top.expect(all);
      if (__ballot(!(all < top.least)) != 0) {
        // which of the lane's logits pass, and those one after the other
        uint32_t pass = 0;
#pragma unroll
        for (int u = 0; u < kLpBatch; ++u)
#pragma unroll
          for (int j = 0; j < kPer; ++j) pass |= !(value_at<T>(raw[u], j) < top.least) ? 1u << (u * kPer + j) : 0u;
        while (__ballot(pass != 0) != 0) {
          const int k = pass != 0 ? __builtin_ctz(pass) : 0, u = k / kPer, j = k % kPer;
          uint4 v = raw[0];
#pragma unroll
          for (int w = 1; w < kLpBatch; ++w) {
            v.x = u == w ? raw[w].x : v.x, v.y = u == w ? raw[w].y : v.y;
            v.z = u == w ? raw[w].z : v.z, v.w = u == w ? raw[w].w : v.w;
          }
          const int step = at + u * kLpWaves, i0 = (step * kWave + lane) * kPer, i = min(i0, a.vocab - kPer) + j;
          top.offer(pass != 0 && step < end && i >= i0 && i >= 0, entry_of(value_of<T>(v, j), (uint32_t)i));
          pass &= pass - 1;
        }
      }
    }
  }
  if constexpr (kTop) {
    top.settle();
    if (lane >= top.count && lane < a.top) bufs[wave][lane] = 0;  // a wave with fewer logits
  }
  s.ones = lane == 0 ? (float)ones : 0.0f;
  s = join_lanes(s);
  if (lane == 0) sums[wave][0] = s.m, sums[wave][1] = s.l, sums[wave][2] = s.x, sums[wave][3] = s.ones;
  __syncthreads();
  {
    float m = sums[0][0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) m = fmaxf(m, sums[w][0]);
    Sums r = {m, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) {
      Sums p = {sums[w][0], sums[w][1], sums[w][2], sums[w][3]};
      rebase(p, m);
      r.l += p.l, r.x += p.x, r.ones += p.ones;
    }
    s = r;
  }
  if constexpr (kTop) {
    // the waves' lists: an entry's place is the number of larger ones in all of them
    const uint64_t mine = lane < a.top ? bufs[wave][lane] : 0;
    int above = 0, at[kLpWaves] = {};
#pragma unroll
    for (int step = kWave; step >= 1; step >>= 1)  // (by halves: the lists are in order)
#pragma unroll
      for (int w = 0; w < kLpWaves; ++w)
        if (at[w] + step <= a.top && bufs[w][at[w] + step - 1] > mine) at[w] += step;
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) above += at[w];
    if (mine != 0 && above < a.top) merged[above] = mine;
    // (a workgroup with fewer logits than n: none of them has the places behind)
    if (tid < a.top) {
      const long long here = min((long long)end * kWave * kPer, (long long)a.vocab) - (long long)first * kWave * kPer;
      if (tid >= here) merged[tid] = 0;
    }
    __syncthreads();
  }
  if (a.splits == 1) {
    write_row<T>(a, row, logits, s, merged, tid);
    return;
  }
  // One of several workgroups of the row: the last to end joins them, in their order.
  const long long at = (long long)row * a.splits + split;
  if (tid == 0) {
    st_coherent(a.part_sums + at * 4, s.m);
    st_coherent(a.part_sums + at * 4 + 1, s.l);
    st_coherent(a.part_sums + at * 4 + 2, s.x);
    st_coherent(a.part_sums + at * 4 + 3, s.ones);
  }
  if (kTop && tid < a.top) __hip_atomic_store(a.part_top + at * a.top + tid, merged[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  wait_stores();
  __syncthreads();
  if (tid == 0) last = atomicAdd(a.count + row, 1) == a.splits - 1;
  __syncthreads();
  if (!last || wave != 0) return;
  if (lane == 0) atomicExch(a.count + row, 0);
  const long long row_at = (long long)row * a.splits;
  Sums p = {kLowest, 0.0f, 0.0f, 0.0f};
  if (lane < a.splits) {
    const float* from = a.part_sums + (row_at + lane) * 4;
    p = {ld_coherent(from), ld_coherent(from + 1), ld_coherent(from + 2), ld_coherent(from + 3)};
  }
  rebase(p, wave_most(p.m));
  p = join_lanes(p);
  if constexpr (kTop) {
    // the lists' first entries, their second ones, and so on, 64 at a time: after the
    // first 64 there is a bound that few of the others pass
    top.start(bufs[0], a.top, lane);
    const uint64_t* from = a.part_top + row_at * a.top;
    const int all = a.splits * a.top;
    for (int base = 0; base < all; base += 4 * kWave) {
      uint64_t e[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int k = base + u * kWave + lane, i = (int)((uint32_t)k * a.per_split >> 20), w = k - i * a.splits;
        e[u] = k < all ? __hip_atomic_load(const_cast<uint64_t*>(from + w * a.top + i), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
      }
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {
        const uint64_t mine = u < 2 ? (u == 0 ? e[0] : e[1]) : (u == 2 ? e[2] : e[3]);
        top.offer(mine != 0, mine);
        if (base + u == 0) top.settle();
      }
    }
    top.settle();
    wave_sync();
  }
  write_row<T>(a, row, logits, p, bufs[0], lane);
}

// Workgroups of a row: about kLpTarget in all, four a CU, with whole batches of vectors
// for every wave (but the row's last: what a batch has past its workgroup's share is
// read and weighed all the same; 5 alternatives of 150 rows of 128256 in bf16 19 us, in
// even shares 24, of 900 rows of 10000 in fp16 19.1 and 19.7).  In even shares, with
// 512, 1024 and 2048, 5 alternatives of 300 rows of 128256 in bf16 took 30, 27 and 32
// us, of 700 rows 46.5, 48.4 and 50.3, of 256 rows of 32000 11.7, 12.0 and 11.9; fewer
// rows have their most in all three.
constexpr int kLpTarget = 1024;
struct Splits {
  int count, each;
};
Splits splits_of(int rows, int vocab, int size) {
  const int steps = (int)(((long long)vocab * size + 16 * kWave - 1) / (16 * kWave)), least = kLpWaves * kLpBatch;
  const int most = std::max(1, std::min({(steps + least - 1) / least, (kLpTarget + rows - 1) / rows, kLpMaxSplits}));
  const int each = ((steps + most - 1) / most + least - 1) / least * least;
  return Splits{(steps + each - 1) / each, each};
}
constexpr int kLpMaxRows = (1 << 24) - 1;  // (a launch has fewer than 2^32 threads in a dimension)

int check_shape(int rows, int vocab, int dtype, int top) {
  if (rows < 0 || rows > kLpMaxRows) return set_error(NSMLP_EINVAL, "rows %d out of range [0, 2^24 - 1]", rows);
  if (vocab < 1 || vocab > (1 << 30)) return set_error(NSMLP_EINVAL, "vocabulary %d out of range [1, 2^30]", vocab);
  if (dtype != NSMLP_DTYPE_F16 && dtype != NSMLP_DTYPE_BF16 && dtype != NSMLP_DTYPE_F32)
    return set_error(NSMLP_EINVAL, "unknown dtype %d", dtype);
  if (top < 0 || top > kLpMaxTop || top > vocab)
    return set_error(NSMLP_EINVAL, "top %d out of range [0, %d], or more than the vocabulary %d", top, kLpMaxTop, vocab);
  return NSMLP_OK;
}
size_t workspace_of(int rows, int vocab, int dtype, int top) {
  const int splits = rows == 0 ? 1 : splits_of(rows, vocab, dtype == NSMLP_DTYPE_F32 ? 4 : 2).count;
  return splits == 1 ? 0 : align_up(kCounterBytes) + (size_t)rows * splits * (16 + 8 * (size_t)top);
}

template <Logit T, bool kTop>
void launch(const LogprobArgs& a, hipStream_t s) {
  const dim3 grid(a.rows, a.splits), block(kLpThreads);
  if (a.vocab >= kPerVector<T>) k_token_logprobs<T, kTop, false><<<grid, block, 0, s>>>(a);
  else k_token_logprobs<T, kTop, true><<<grid, block, 0, s>>>(a);
}
template <Logit T>
void launch(const LogprobArgs& a, hipStream_t s) {
  a.top > 0 ? launch<T, true>(a, s) : launch<T, false>(a, s);
}

}  // namespace

}  // namespace nsmlp

using namespace nsmlp;

extern "C" {

size_t nsmlp_token_logprobs_workspace_bytes(int rows, int vocab, int dtype, int top) {
  return check_shape(rows, vocab, dtype, top) ? 0 : workspace_of(rows, vocab, dtype, top);
}

int nsmlp_token_logprobs(const void* logits, long long row_stride, int dtype, int rows, int vocab, const int64_t* tokens, int top,
                         float* logprob, float* entropy, int64_t* top_ids, float* top_logprobs, void* ws, size_t ws_bytes,
                         void* stream) {
  NSMLP_FAULT_POINT("token_logprobs");
  int rc = check_shape(rows, vocab, dtype, top);
  if (rc || rows == 0) return rc;
  if ((tokens == nullptr) != (logprob == nullptr)) return set_error(NSMLP_EINVAL, "tokens and logprob go together");
  if (top > 0 && (top_ids == nullptr || top_logprobs == nullptr))
    return set_error(NSMLP_EINVAL, "top_ids and top_logprobs must be non-NULL");
  const int size = dtype == NSMLP_DTYPE_F32 ? 4 : 2;
  if (logits == nullptr || (uintptr_t)logits % size != 0)
    return set_error(NSMLP_EINVAL, "logits must be non-NULL and aligned to their elements");
  const size_t need = workspace_of(rows, vocab, dtype, top);
  if (need > 0 && (ws == nullptr || ws_bytes < need))
    return set_error(NSMLP_ENOSPC, "token_logprobs workspace needs %zu bytes, got %zu", need, ws == nullptr ? (size_t)0 : ws_bytes);
  if (need > 0 && ((uintptr_t)ws & (kAlign - 1)) != 0) return set_error(NSMLP_EINVAL, "workspace must be 256-byte aligned");
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return set_error(NSMLP_ENODEV, "no HIP device");
  LogprobArgs a = {};
  a.logits = (const uint8_t*)logits;
  a.row_bytes = row_stride * size;
  a.rows = rows, a.vocab = vocab, a.top = top;
  const Splits s = splits_of(rows, vocab, size);
  a.splits = s.count, a.each = s.each, a.per_split = ((1u << 20) + s.count - 1) / s.count;
  a.tokens = tokens;
  a.logprob = logprob, a.entropy = entropy;
  a.top_ids = top_ids, a.top_logprobs = top_logprobs;
  if (need > 0) {
    a.part_top = (uint64_t*)((char*)ws + align_up(kCounterBytes));
    a.part_sums = (float*)(a.part_top + (size_t)rows * a.splits * top);
    a.count = (int*)((char*)ws + kBlkCountOff);
  }
  if (dtype == NSMLP_DTYPE_F16) launch<Logit::kF16>(a, (hipStream_t)stream);
  else if (dtype == NSMLP_DTYPE_BF16) launch<Logit::kBf16>(a, (hipStream_t)stream);
  else launch<Logit::kF32>(a, (hipStream_t)stream);
  return check_launch("nsmlp_token_logprobs");
}

}  // extern "C"
