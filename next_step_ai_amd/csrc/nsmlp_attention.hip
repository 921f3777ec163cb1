// Attention over the paged 8-bit K/V cache (layouts: nsmlp_kv.h).
//
// For a query row and the keys j it sees, with codes k, v, scales ks, vs of
// the key's (block, head) and c = softmax scale * log2(e):
//   s_j = c ks_j (q . k_j)             the score, in powers of two
//   o   = sum_j 2^s_j vs_j v_j / sum_j 2^s_j
// The V scale goes into the exponent: with e_j = s_j + log2(vs_j) and a
// reference m near the largest e_j,
//   acc = sum_j 2^(e_j - m) v_j,   l = sum_j 2^(e_j - m) / vs_j,   o = acc / l
// so a weight costs one fused multiply-add and one exp2, the weights fit fp16
// whatever the scales of the blocks are, and the codes enter the products
// exactly.  m follows the running maximum lazily: when it is set, the largest
// weight is about 2^10, and it is set again only where the weights' sums (of 4
// or 8, kept anyway) pass 2^15.  So most tiles neither look for a maximum nor
// rescale acc, no weight leaves fp16, and weights down to 2^-24 of the largest
// keep their 11 bits (with the largest at 1 those below 2^-14 lost some, and
// outputs over thousands of keys half a rounding).  m is an integer, so that
// rescaling is exact.  acc, l, m and the scores are fp32.  A weight is an operand
// of the products in two fp16 parts where rows are few, and rounded to fp16
// once where they are many, as a second product would cost as much as the first.
// There l takes it as rounded: where few keys carry a row its rounding cancels.
// A block whose V scale is far below the others' (its V are zeros, say) has
// weights that fp16 rounds to nothing, though its keys' share of l is as large as
// any: weights whose sum is small enter l as they are.
#include <mutex>
#include <type_traits>

#include "nsmlp_kv.h"

namespace nsmlp {

namespace {

constexpr float kLowest = -3.402823466e38f;
constexpr float kSumLimit = 32768.0f;
constexpr float kLift = 10.0f;
constexpr int kUnitLog2 = 15;
constexpr float kUnit = 1.0f / (1 << kUnitLog2);
// Sums of weights below this may hold subnormal ones, which lose bits: above, what
// 8 weights lose is below 2^-16 of the sum.
constexpr float kSmallSum = 0.015625f;

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

__device__ __forceinline__ half8_t join4(uint2 a, uint2 b) {
  return as_h8(uint4{a.x, a.y, b.x, b.y});
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const half2_t h = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(uint32_t, h);
}

template <bool kBf16>
__device__ __forceinline__ uint16_t to_out(float x) {
  if constexpr (kBf16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  else return f2h(x);
}

// bf16 queries become fp16 under a power of two of the row's own: its largest
// magnitude (bits `top`) lands in [1, 2), what it loses is below 2^-24 of that.
__device__ __forceinline__ int row_exponent(uint32_t top) { return min(max((int)(top >> 7), 1), 254) - 127; }

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__device__ __forceinline__ uint4 bf16_to_f16(const uint4& raw, int e) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = word(raw, i);
    o[i] = pack_f16(ldexpf(__uint_as_float(w << 16), -e), ldexpf(__uint_as_float(w & 0xFFFF0000u), -e));
  }
  return uint4{o[0], o[1], o[2], o[3]};
}

// Scores beyond 2^12 (in powers of two).  s + lv - m in one fused operation needs
// lv - m rounded first, which costs the weight 2^-24 |m|, and past 2^27 the
// difference of two roundings of a score leaves exp2's range.  So where m is that
// far, a score is rounded, m subtracted from it, which is exact where the two
// are close, and lv added then.  Such an m is the largest s + lv, rounded; what
// that rounding leaves above it is 2^4 for scores below 2^28, and more only where
// lv, too, is beyond the score's last bit: such weights count as 2^15.
constexpr float kFar = 4096.0f;

__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= kFar && m != kLowest; }

// the reference that a row whose largest s + lv is `top` wants: a whole number
__device__ __forceinline__ float reference_of(float top) {
  const float c = ceilf(top);
  return is_far(c) ? c : c - kLift;
}
__device__ __forceinline__ float far_exponent(float s, float g, float lv, float m) {
#pragma clang fp contract(off)
  const float t = s * g;
  return is_far(m) ? fminf((t - m) + lv, 15.0f) : (t - m) + lv;
}

// Pages of a range of keys, held one per lane: 64 pages from page `first`.
struct Pages {
  uint32_t lo, hi;   // where the (block, head)'s codes start (block 0's where the entry is not a block)
  float ks, lv, iv;  // K scale, log2 of the V scale, kUnit over it
  unsigned long long bad;
  int first;
};

__device__ __forceinline__ Pages load_pages(const KvAttnArgs& a, int req, int h, int first, int last, int lane) {
  Pages p;
  p.first = first;
  const int pg = min(min(first + lane, last), a.max_blocks - 1);
  const int id = a.table[(long long)req * a.max_blocks + pg];
  const bool ok = id >= 0 && id < a.c.num_blocks;
  const long long bh = (long long)(ok ? id : 0) * a.c.heads + h;
  const long long off = bh * (2 * a.c.B * a.c.D);
  p.lo = (uint32_t)off, p.hi = (uint32_t)(off >> 32);
  const float2 s = *reinterpret_cast<const float2*>(a.c.scale + bh * 2);
  const float sv = s.y == 0.0f ? kKvScaleMin : s.y;  // a block that nothing was stored in
  p.bad = __ballot(!ok);
  p.ks = s.x;
  p.lv = log2_fast(sv);
  p.iv = kUnit / sv;
  return p;
}

__device__ __forceinline__ const uint8_t* page_data(const KvAttnArgs& a, const Pages& p, int i) {
  return a.c.data + ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)p.lo, i) |
                     (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)p.hi, i) << 32);
}

__device__ __forceinline__ float lane_of(float v, int i) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
}

// What a row's acc is multiplied by, and its lse, at the end.
__device__ __forceinline__ float inverse_of(float l) { return l == 0.0f ? 0.0f : kUnit / l; }
__device__ __forceinline__ float lse_of(float m, float x) {
  return x == 0.0f ? -INFINITY : (m + (float)kUnitLog2 + log2f(x)) * 0.6931471805599453f;
}

// Whether token i of the step is there.  (Lengths whose sum passes 32 bits leave
// requests' first tokens below zero.)
__device__ __forceinline__ bool in_step(const KvAttnArgs& a, int i) { return (unsigned)i < (unsigned)a.total; }

// A unit in scalar registers (left in memory it would be read again after
// every barrier).
__device__ __forceinline__ KvUnit load_unit(const KvUnit* p) {
  const KvUnit v = *p;
  return KvUnit{uniform(v.req),  uniform(v.row),   uniform(v.kv_begin), uniform(v.kv_end),
                uniform(v.part), uniform(v.first), uniform(v.parts),    0};
}

// ---------------------------------------------------------------- stream --
// Up to 16 query rows against a range of keys.  The workgroup's waves share a
// unit's keys out and their results meet in LDS; products with the keys (or
// dims) as rows and the queries as columns, so that a column's weights leave the
// first product where the second wants them.
//
// What bounds it: the codes' way from HBM, read once.  All K/V heads' requests
// together are cut into one equal share per CU, so that uneven lengths cost
// nothing, and a wave has the next 32 keys' codes in flight while it works on
// 32: 64 uneven requests (429 MB) 82 us, 5.2 TB/s; one token over 131000 keys
// (269 MB, 31 partial results per row to join) 57.5 us, 4.7 TB/s.  A short chat (777
// keys) takes 9.5 us, most of it the chain launch, schedule, lengths, block
// table, scales, codes, join.
template <int D, int NW>
struct StreamLds {
  float sum[NW][16][D + 4];  // the waves' results
  float ml[NW][2][16];
  int last;
};

template <int D>
struct StreamTile {  // 32 keys, two tiles of 16: codes, and their blocks' scales in scalar registers
  uint4 k[2][D / 64], v[2][D / 64];
  float ks[2], lv[2], iv[2];
  int bad;
};

__device__ __forceinline__ void st_coherent2(float* p, float a, float b) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32,
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 ld_coherent2(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<uint64_t*>(const_cast<float*>(p)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Zeros and -inf in the rows of a request without keys (a refused one), which
// may be more than a unit's 16.
template <int D>
__device__ __forceinline__ void fill_unseen(const KvAttnArgs& a, int req, int h) {
  const int q0 = uniform(a.q_start[req]), q_len = uniform(a.q_start[req + 1]) - q0;
  const long long first = max(q0, 0), tokens = min((long long)q0 + q_len, (long long)a.total) - first;
  const int pieces = a.group * D / 8;  // of a token, 16 bytes each
  for (long long i = threadIdx.x; i < tokens * pieces; i += blockDim.x)
    reinterpret_cast<uint4*>(a.out + ((first + i / pieces) * a.c.heads + h) * a.group * D)[i % pieces] = uint4{0, 0, 0, 0};
  if (a.lse == nullptr) return;
  for (long long i = threadIdx.x; i < tokens * a.group; i += blockDim.x)
    a.lse[((first + i / a.group) * a.c.heads + h) * a.group + i % a.group] = -INFINITY;
}

template <int D, int kFmt, bool kBf16, int NW>
__device__ __forceinline__ void stream_unit(const KvAttnArgs& a, const KvUnit u, int h, StreamLds<D, NW>& lds) {
  constexpr int NJ = D / 64, KS = D / 32, ND = D / 16;
  // Weights go in two fp16 parts, 22 bits, so that their rounding does not add to
  // the output's own (fp16: error against 64 bits 2.9e-4 -> 2.1e-4 of the norm, one
  // rounding; bf16: 64 requests' outputs 7.6e-4 -> 5e-5 from those of fp32 weights).
  // The products have the time, as the codes' way from memory takes longer:
  // 131000 keys 57.8 us with one part and with two, 64 requests 82.7 and 82.9.
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int q0 = uniform(a.q_start[u.req]), q_len = uniform(a.q_start[u.req + 1]) - q0, kv_len = uniform(a.kv_len[u.req]);
  const int rows = q_len > kKvRowsA ? kKvRowsA : min(q_len * a.group, kKvRowsA);

  // this wave's keys
  const int each = ((u.kv_end - u.kv_begin + NW - 1) / NW + 31) & ~31;
  const int begin = u.kv_begin + wave * each, end = min(begin + each, u.kv_end);
  const int last = max(0, (u.kv_end - 1) >> a.c.b_shift);

  // the first tiles' codes are on their way while the queries are made ready
  unsigned long long bad_seen = 0;
  Pages pages;
  const auto load = [&](StreamTile<D>& t, int pos) {
    t.bad = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = pos + 16 * s, pg = min(at >> a.c.b_shift, last) - pages.first;
      t.ks[s] = lane_of(pages.ks, pg), t.lv[s] = lane_of(pages.lv, pg), t.iv[s] = lane_of(pages.iv, pg);
      t.bad |= ((int)(pages.bad >> pg) & 1) << s;
      const uint8_t* kb = page_data(a, pages, pg) + ((at & (a.c.B - 1)) >> 4) * (16 * D);
      const uint8_t* vb = kb + a.c.B * D;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        t.k[s][j] = *reinterpret_cast<const uint4*>(kb + j * 1024 + lane * 16);
        t.v[s][j] = *reinterpret_cast<const uint4*>(vb + j * 1024 + lane * 16);
      }
    }
  };
  // past the wave's keys its last tile is read again: no branch around a load
  const int last_tile = begin < end ? begin + ((end - 1 - begin) & ~31) : begin;
  const auto fetch = [&](StreamTile<D>& t, int pos) {
    pos = min(pos, last_tile);
    if (min((pos + 31) >> a.c.b_shift, last) - pages.first >= kWave) {
      pages = load_pages(a, u.req, h, pos >> a.c.b_shift, last, lane);
      bad_seen |= pages.bad;
    }
    load(t, pos);
  };
  StreamTile<D> t0, t1;
  if (begin < end) {
    pages = load_pages(a, u.req, h, begin >> a.c.b_shift, last, lane);
    bad_seen = pages.bad;
    load(t0, begin);
  }

  // queries: columns of the products, 8 dims per lane and step
  half8_t q[KS];
  float rowf = a.scale_log2;
  const int tok = col / a.group;
  const bool in = col < rows && in_step(a, q0 + tok);
  const int limit = in ? kv_len - q_len + tok + 1 : 0x7FFFFFFF;  // keys that the row sees
  {
    const uint16_t* src = a.q + (long long)(q0 + tok) * a.q_row + (long long)(h * a.group + col % a.group) * a.q_head;
    uint4 raw[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s)
      raw[s] = in ? *reinterpret_cast<const uint4*>(src + 64 * (s >> 1) + 16 * grp + 8 * (s & 1)) : uint4{0, 0, 0, 0};
    if constexpr (kBf16) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(word(raw[s], i) & 0x7FFFu, (word(raw[s], i) >> 16) & 0x7FFFu));
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, kWave));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, kWave));
      const int e = row_exponent(top);
      rowf *= ldexpf(1.0f, e);
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = as_h8(bf16_to_f16(raw[s], e));
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = as_h8(raw[s]);
    }
  }
  // keys below this need no mask: every row of the unit sees them
  const int plain = kv_len - q_len + 1;

  float m = kLowest, l = 0.0f;  // reference, sum of the weights
  float sum_limit = kSumLimit;  // (below any sum where m is far)
  float4_t acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

  const auto use = [&](auto masked, const StreamTile<D>& t, int pos) {
    constexpr bool kMasked = decltype(masked)::value;
    float4_t sc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        sc[s] = mfma16(join4(kv_half4<kFmt>(word(t.k[s][i >> 1], 2 * (i & 1))), kv_half4<kFmt>(word(t.k[s][i >> 1], 2 * (i & 1) + 1))),
                       q[i], sc[s]);
    mfma_drain();
    // bit 4 s + i: whether the row sees the lane's key i of the s-th 16
    uint32_t see = 0xFF;
    if constexpr (kMasked) {
      see = 0;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int n = (t.bad >> s) & 1 ? 0 : min(max(limit - pos - 16 * s - 4 * grp, 0), 4);
        see |= ((1u << n) - 1u) << (4 * s);
      }
    }
    uint2 w[2], rest[2];  // weights, and what their rounding left
    float dl;
    float gs[2] = {t.ks[0] * rowf, t.ks[1] * rowf}, lvs[2] = {t.lv[0], t.lv[1]};
    const auto weights = [&]() {
      float sums[2];
      dl = 0.0f;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const float g = gs[s], c = lvs[s] - m;
        float p[4], share = t.iv[s];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = exp2_fast(__builtin_fmaf(sc[s][i], g, c));
        if constexpr (kMasked) {
          // a hidden key's weight is zero whatever its block's scales are
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = (see >> (4 * s + i)) & 1 ? p[i] : 0.0f;
          share = (see >> (4 * s)) & 0xF ? share : 0.0f;
        }
        w[s] = uint2{pack_f16(p[0], p[1]), pack_f16(p[2], p[3])};
        const half2_t a0 = as_half2(w[s].x), a1 = as_half2(w[s].y);
        rest[s] = uint2{pack_f16(p[0] - (float)a0.x, p[1] - (float)a0.y), pack_f16(p[2] - (float)a1.x, p[3] - (float)a1.y)};
        sums[s] = (p[0] + p[1]) + (p[2] + p[3]);
        dl = __builtin_fmaf(sums[s], share, dl);
      }
      return fmaxf(sums[0], sums[1]);
    };
    const float sum = weights();
    if (__builtin_expect_with_probability(__any(sum > sum_limit), 0, 0.999)) {
      float top = kLowest;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, (see >> (4 * s + i)) & 1 ? __builtin_fmaf(sc[s][i], gs[s], lvs[s]) : kLowest);
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = reference_of(fmaxf(top, __shfl_xor(top, 32, kWave)));
      top = fmaxf(m, top);  // (never down: other rows may have asked)
      const float scale = exp2_fast(m - top);
      m = top;
      sum_limit = is_far(m) ? -1.0f : kSumLimit;
      l *= scale;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] *= scale;
      if (__builtin_expect_with_probability(__any(is_far(m)), 0, 0.999)) {  // the scores become their weights' exponents
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[s][i] = far_exponent(sc[s][i], gs[s], lvs[s], m);
          gs[s] = 1.0f, lvs[s] = m;
        }
      }
      (void)weights();
    }
    l += dl;
    uint32_t keep[2] = {~0u, ~0u};
    if (kFmt == NSMLP_KV_E4M3 && kMasked) {
      // codes past the end may be NaNs: a zero weight does not hide them
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int left = (t.bad >> s) & 1 ? 0 : kv_len - (pos + 16 * s + 4 * grp);
        keep[s] = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
      }
    }
    const half8_t wh = join4(w[0], w[1]), wr = join4(rest[0], rest[1]);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const half8_t v = join4(kv_half4<kFmt>(word(t.v[0][d >> 2], d & 3) & keep[0]), kv_half4<kFmt>(word(t.v[1][d >> 2], d & 3) & keep[1]));
      acc[d] = mfma16(v, wh, acc[d]);
      acc[d] = mfma16(v, wr, acc[d]);
    }
  };
  if (begin < end) {
    int pos = begin;
    while (pos + 64 <= min(end, plain) && bad_seen == 0) {  // two tiles, the next two's codes behind them
      fetch(t1, pos + 32);
      if (bad_seen != 0) break;  // (of a new window of pages, which may be t1's)
      use(std::false_type{}, t0, pos);
      fetch(t0, pos + 64);
      use(std::false_type{}, t1, pos + 32);
      pos += 64;
    }
    while (pos < end) {
      fetch(t1, pos + 32);
      use(std::true_type{}, t0, pos);
      t0 = t1;
      pos += 32;
    }
  }
  if (bad_seen != 0 && lane == 0) atomicOr(a.status, NSMLP_STATUS_BLOCK_UNAVAILABLE);

  mfma_drain();
  // join the waves: each result under the largest reference
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (grp == 0) lds.ml[wave][0][col] = m, lds.ml[wave][1][col] = l;
  __syncthreads();
  {
    float top = kLowest;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, lds.ml[w][0][col]);
    const float scale = exp2_fast(m - top);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4_t*>(&lds.sum[wave][col][64 * j + 16 * grp + 4 * i]) =
            float4_t{acc[4 * j][i], acc[4 * j + 1][i], acc[4 * j + 2][i], acc[4 * j + 3][i]} * scale;
  }
  __syncthreads();
  constexpr int kPerRow = NW * kWave / 16, kDims = D / kPerRow;
  const int row = tid / kPerRow, d0 = tid % kPerRow * kDims;
  float mr = kLowest, lr = 0.0f, o[kDims] = {};
#pragma unroll
  for (int w = 0; w < NW; ++w) mr = fmaxf(mr, lds.ml[w][0][row]);
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float f = exp2_fast(lds.ml[w][0][row] - mr);
    lr += lds.ml[w][1][row] * f;
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] += lds.sum[w][row][d0 + d];
  }
  if (u.part >= 0) {
    // One of several units of these rows: eight at a time are added up by the
    // last of them to end, their sums again eight at a time, and so on, each
    // sum in the order of the parts, so that the result does not depend on who
    // is last.  A level costs one write, one atomic and one read that all
    // threads have in flight at once (4 us; one workgroup reading 64 partials
    // of 8 KB took 20 us).
    int idx = u.part - u.first, n = u.parts, stride = 1;
    int* count = a.count;
    while (n > 1) {
      const int group = idx >> 3, size = min(8, n - 8 * group);
      if (size > 1) {
        const long long step = (long long)stride * a.c.heads * kKvRowsA;
        const long long at = ((long long)u.first * a.c.heads + h) * kKvRowsA + row + idx * step;
        if (row < rows) {
#pragma unroll
          for (int d = 0; d < kDims; d += 2) st_coherent2(a.acc_a + at * D + d0 + d, o[d], o[d + 1]);
          if (d0 == 0) st_coherent2(a.ml_a + 2 * at, mr, lr);
        }
        wait_stores();
        __syncthreads();
        int* arrived = count + (u.first + group * 8 * stride) * a.c.heads + h;
        if (tid == 0) lds.last = atomicAdd(arrived, 1) == size - 1;
        __syncthreads();
        if (!lds.last) return;
        if (tid == 0) atomicExch(arrived, 0);
        if (row < rows) {
          const long long from = at + (group * 8 - idx) * step;
          float2 ml[8], y[8][kDims / 2];
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const long long q_at = from + min(p, size - 1) * step;  // (the last again: no branch between the reads)
            ml[p] = ld_coherent2(a.ml_a + 2 * q_at);
#pragma unroll
            for (int d = 0; d < kDims / 2; ++d) y[p][d] = ld_coherent2(a.acc_a + q_at * D + d0 + 2 * d);
          }
          mr = ml[0].x;
#pragma unroll
          for (int p = 1; p < 8; ++p) mr = fmaxf(mr, ml[p].x);
          lr = 0.0f;
#pragma unroll
          for (int d = 0; d < kDims; ++d) o[d] = 0.0f;
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const float f = exp2_fast(ml[p].x - mr);
            if (p < size) {
              lr += ml[p].y * f;
#pragma unroll
              for (int d = 0; d < kDims / 2; ++d) o[2 * d] += y[p][d].x * f, o[2 * d + 1] += y[p][d].y * f;
            }
          }
        }
      }
      idx = group, n = (n + 7) >> 3, stride *= 8;
      count += kKvCounters;  // each level has counters of its own
    }
  }
  if (row < rows) {
    const int tok_r = q0 + row / a.group, head = h * a.group + row % a.group;
    if (in_step(a, tok_r)) {
      const float inv = inverse_of(lr);
      const long long at = (long long)tok_r * a.c.heads * a.group + head;
#pragma unroll
      for (int d = 0; d < kDims; d += 2)
        *reinterpret_cast<uint32_t*>(a.out + at * D + d0 + d) =
            to_out<kBf16>(o[d] * inv) | (uint32_t)to_out<kBf16>(o[d + 1] * inv) << 16;
      if (a.lse != nullptr && d0 == 0) a.lse[at] = lse_of(mr, lr);
    }
  }
}

// A workgroup's share of list a: the units from the share's first to the next
// one's.  The 8 XCDs take shares in turn and all heads of a share: heads of a
// block have their scales in one line, which one L2 then fetches once.
template <int D, int kFmt, bool kBf16, int NW>
__device__ __forceinline__ void stream_share(const KvAttnArgs& a, int block, StreamLds<D, NW>& lds) {
  const int h = (block >> 3) % a.c.heads, share = (block >> 3) / a.c.heads * 8 + (block & 7);
  const int shares = min(a.sched[1], a.s.shares), units = min(a.sched[0], a.s.max_units_a);
  if (share >= shares) return;
  const int32_t* start = a.sched + a.s.off_shares;
  const int end = share + 1 < shares ? min(start[share + 1], units) : units;
  const KvUnit* list = reinterpret_cast<const KvUnit*>(a.sched + a.s.off_units_a);
  for (int i = start[share]; i < end; ++i) {
    const KvUnit u = load_unit(list + i);
    if (u.kv_end == 0) fill_unseen<D>(a, u.req, h);
    else stream_unit<D, kFmt, kBf16, NW>(a, u, h, lds);
    __syncthreads();
  }
}

template <int D, int kFmt, bool kBf16>
__global__ void __launch_bounds__(4 * kWave) k_attn_stream(KvAttnArgs a) {
  kernarg_warm<sizeof(KvAttnArgs)>();
  __shared__ __attribute__((aligned(16))) StreamLds<D, 4> lds;
  stream_share<D, kFmt, kBf16, 4>(a, blockIdx.x, lds);
}

// ----------------------------------------------------------------- tiles --
// Prompts and chunks: NW waves of 32 query rows each against tiles of 64 keys
// that the workgroup decodes to fp16 once, in LDS, as the operands of
// v_mfma_f32_32x32x16_f16 (A rows: keys or dims, B columns: queries).  Codes
// are taken 16 bytes at a time from two places, a dword of each makes a lane's
// 8 operands, of K and of V alike:
//   K fragment (32 keys, 16 dims): lane l: key l % 32, dims 16 g + 4 i + 0..3 and D / 2 + the same
//   V fragment (32 dims, 16 keys): lane l: keys 4 h + 0..3 and 8 + 4 h + 0..3, h = l / 32
// The scores of a query stay in its two lanes, in the order in which the
// second product wants the weights.
//
// What bounds it: the matrix cores, and the vector work that does not hide
// behind them (an exp2, a multiply-add and a conversion per weight, and the
// decoding, shared by 128 or 256 rows).  A product follows another after about
// 47 cycles instead of 32, half of a step with 8 waves is the wave's own vector
// half, in which the SIMD's other wave has its products: 2048 tokens over 14336
// cached, 128 heads of 128, 2.0 ms, 1.03 PFLOP/s, matrix cores busy 54%; a
// prompt of 4000 tokens and 32 heads 165-180 us (0.73-0.79 PFLOP/s: 1000 tiles
// of uneven length on 512 places).
constexpr int kTileKeys = 64;

__device__ __forceinline__ float max8(const float16_t& s, int at) {
  return fmaxf(fmaxf(fmaxf(s[at], s[at + 1]), fmaxf(s[at + 2], s[at + 3])),
               fmaxf(fmaxf(s[at + 4], s[at + 5]), fmaxf(s[at + 6], s[at + 7])));
}

// What the weights of 16 keys need to know of their block: K scale, log2 of
// the V scale, kUnit over it, and (as bits) whether it is no block.
typedef float4_t TileMeta;

template <int D>
constexpr int kTileBytes = (D / 16 * 2 + D / 32 * 4) * 1024;  // fragments of a tile, 1 KB each
template <int D>
constexpr int kTileLds = 2 * kTileBytes<D> + 4 * 4 * (int)sizeof(TileMeta);

template <int D, int kFmt, bool kBf16, int NW, bool kLse>
__device__ __forceinline__ void tile_unit(const KvAttnArgs& a, const KvUnit u, int h, char* lds) {
  constexpr int KS = D / 16, ND = D / 32, kRows = 32 * NW;
  constexpr int kKBytes = 2 * KS * 1024, kVBytes = 4 * ND * 1024;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  TileMeta* const metas = reinterpret_cast<TileMeta*>(lds + 2 * kTileBytes<D>);
  const int q0 = uniform(a.q_start[u.req]), q_len = uniform(a.q_start[u.req + 1]) - q0, kv_len = uniform(a.kv_len[u.req]);
  const int rows = min(q_len * a.group - u.row, kRows);
  const int r = wave * 32 + col, row = u.row + r, tok = row / a.group;
  const bool in = r < rows && in_step(a, q0 + tok);
  const int limit = in ? kv_len - q_len + tok + 1 : 0x7FFFFFFF;  // keys that the row sees
  const int last = max(0, (u.kv_end - 1) >> a.c.b_shift);
  const int tiles = (u.kv_end - u.kv_begin + kTileKeys - 1) / kTileKeys;

  // The 16 keys of a tile that this wave decodes: with 8 waves K (lower four)
  // or V, with 4 both.  Where its lane reads in a (block, head)'s 16 keys, and
  // where it writes.
  constexpr int kRoles = NW == 8 ? 1 : 2;
  const int part = wave & 3;
  const bool upper = NW == 8 && wave >= 4;
  uint32_t src[kRoles], src2[kRoles];
  int dst[kRoles], dst_step[kRoles];
#pragma unroll
  for (int o = 0; o < kRoles; ++o) {
    const bool v = kRoles == 2 ? o == 1 : upper;
    if constexpr (D == 128) {
      const int g = lane >> 4, t = lane & 15;
      src[o] = v ? a.c.B * D + (g & 1) * 1024 + half * 256 + t * 16 : lane * 16;
      src2[o] = src[o] + (v ? 512 : 1024);
      dst[o] = v ? kKBytes + (part * ND * 64 + lane) * 16
                 : ((((part >> 1) * KS + (g >> 1)) * 64) + (g & 1) * 32 + (part & 1) * 16 + t) * 16;
      dst_step[o] = v ? 1024 : 2048;
    } else {  // (the upper lanes repeat the lower ones)
      const int g = (lane >> 4) & 1, t = lane & 15;
      src[o] = (v ? a.c.B * D : 0) + g * 256 + t * 16;
      src2[o] = src[o] + 512;
      dst[o] = v ? kKBytes + (part * ND * 64 + g * 32 + t) * 16 : (((part >> 1) * KS * 64) + g * 32 + (part & 1) * 16 + t) * 16;
      dst_step[o] = 1024;
    }
  }
  unsigned long long bad_seen = 0;
  Pages pages = load_pages(a, u.req, h, u.kv_begin >> a.c.b_shift, last, lane);
  if (tiles > 0) bad_seen = pages.bad;
  // whether V scales so far lie more than a factor of 2^4 from the first one: only
  // then can a weight that matters to l be too small for fp16 (the largest is
  // 2^10, and weights below 2^-27 of it are lost at most)
  const float lv_first = lane_of(pages.lv, 0);
  const auto apart = [&]() { return __ballot(!(fabsf(pages.lv - lv_first) <= 4.0f)); };
  unsigned long long uneven = apart();
  // this wave's page in tile i, as a lane of `pages`; past the last tile again the last
  const auto at_of = [&](int i) { return u.kv_begin + min(i, tiles - 1) * kTileKeys + 16 * part; };
  const auto page_of = [&](int i) { return min(at_of(i) >> a.c.b_shift, last) - pages.first; };
  uint4 raw[kRoles][2];
  const auto fetch = [&](int o, int i) {
    const int at = at_of(i);
    const uint8_t* base = page_data(a, pages, page_of(i)) + ((at & (a.c.B - 1)) >> 4) * (16 * D);
    raw[o][0] = *reinterpret_cast<const uint4*>(base + src[o]);
    raw[o][1] = *reinterpret_cast<const uint4*>(base + src2[o]);
  };
  // one of the 8 dwords at a time: decoded (half 0, 1 of piece j), and written with its pair
  uint2 lo_piece;
  const auto decode = [&](int o, int i, char* buf, int step) {
    const int j = step >> 1;
    uint32_t w = word(raw[o][step & 1], j);
    if (kFmt == NSMLP_KV_E4M3 && (kRoles == 2 ? o == 1 : true)) {
      // V codes past the end may be NaNs: a zero weight does not hide them
      // (with 8 waves the lower four, which have K, keep all)
      const int left = kv_len - (at_of(i) + 8 * (step & 1) + 4 * (D == 128 ? half : (lane >> 4) & 1));
      const bool bad = (pages.bad >> page_of(i)) & 1;
      const uint32_t mask = bad || left <= 0 ? 0u : left >= 4 ? ~0u : (1u << (8 * left)) - 1u;
      w &= kRoles == 2 || upper ? mask : ~0u;
    }
    const uint2 v = kv_half4<kFmt>(w);
    if (!(step & 1)) {
      lo_piece = v;
    } else {
      int to = dst[o] + j * dst_step[o];
      if constexpr (D == 64) {
        // V: dims 4 t + j are rows t + 16 (j % 2) of fragment j / 2
        if (kRoles == 2 ? o == 1 : upper) to = dst[o] + (j >> 1) * 1024 + (j & 1) * 256;
      }
      *reinterpret_cast<uint4*>(buf + to) = uint4{lo_piece.x, lo_piece.y, v.x, v.y};
    }
  };
  const auto store_meta = [&](int i) {  // (every lane the same, and both waves of a part)
    const int pg = page_of(i);
    metas[(i & 3) * 4 + part] = TileMeta{lane_of(pages.ks, pg), lane_of(pages.lv, pg), lane_of(pages.iv, pg),
                                         __int_as_float((int)((pages.bad >> pg) & 1))};
  };
  // the window of pages moves before the first tile that is not all in it is
  // fetched, and keeps tiles from `from` on
  const auto window_end = [&]() {  // that tile
    const int keys = ((pages.first + kWave) << a.c.b_shift) - u.kv_begin;
    return pages.first + kWave > last ? 0x7FFFFFFF : keys / kTileKeys;
  };
  int turn_at = window_end();
  const auto turn_pages = [&](int from, int need) {
    if (__builtin_expect_with_probability(need >= turn_at, 0, 0.95)) {
      pages = load_pages(a, u.req, h, (u.kv_begin + min(from, tiles - 1) * kTileKeys) >> a.c.b_shift, last, lane);
      bad_seen |= pages.bad;
      uneven |= apart();
      turn_at = window_end();
    }
  };
  if (tiles > 0) {
#pragma unroll
    for (int o = 0; o < kRoles; ++o) fetch(o, 0);
  }

  half8_t q[KS];
  float rowf = a.scale_log2;
  {
    const uint16_t* from = a.q + (long long)(q0 + tok) * a.q_row + (long long)(h * a.group + row % a.group) * a.q_head;
    uint4 part_q[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // dims of K fragment s in this half of the wave
      const int d = D == 128 ? 16 * (2 * (s & 1) + half) + 4 * (s >> 1) : 16 * half + 4 * s;
      uint2 lo = {0, 0}, hi = {0, 0};
      if (in) lo = *reinterpret_cast<const uint2*>(from + d), hi = *reinterpret_cast<const uint2*>(from + d + D / 2);
      part_q[s] = uint4{lo.x, lo.y, hi.x, hi.y};
    }
    if constexpr (kBf16) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(word(part_q[s], i) & 0x7FFFu, (word(part_q[s], i) >> 16) & 0x7FFFu));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, kWave));
      const int e = row_exponent(top);
      rowf *= ldexpf(1.0f, e);
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = as_h8(bf16_to_f16(part_q[s], e));
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = as_h8(part_q[s]);
    }
  }
  // keys below this need no mask in this wave
  const int plain = kv_len - q_len + (u.row + min(wave * 32, rows)) / a.group + 1;

  float m = kLowest, l = 0.0f, x = 0.0f;
  float sum_limit = kSumLimit;  // (below any sum where m is far)
  float16_t acc[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[n][e] = 0.0f;

  // Matrix half of a step: the product of the weights before with their
  // values, and the scores of a tile, one product after the other.  Operands
  // are fetched 6 products ahead, as an LDS read takes as long as several of
  // them, and `side(k)` goes behind the k-th product: a wave issues in order,
  // and a product keeps the matrix core for 32 cycles in which the wave can
  // issue 7 other instructions.
  constexpr int kValues = 4 * ND, kAll = kValues + 2 * KS, kAhead = 6;
  float16_t s[2];
  uint4 w[4];
  const auto matrix = [&](const char* vbuf, const char* kbuf, auto both, auto&& side) {
    constexpr int kSteps = decltype(both)::value ? kAll : kValues;
    const half8_t* vf = reinterpret_cast<const half8_t*>(vbuf + kKBytes) + lane;
    const half8_t* kf = reinterpret_cast<const half8_t*>(kbuf) + lane;
    half8_t ring[8];
    const auto get = [&](int k) {  // values: 16 keys' weights times all dims; scores: a fragment of either 32 keys
      ring[k & 7] = k < kValues ? vf[k * 64] : kf[((k & 1) * KS + ((k - kValues) >> 1)) * 64];
    };
    sched_fence();
#pragma unroll
    for (int k = 0; k < kAhead; ++k) get(k);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      sched_fence();
      if (k + kAhead < kSteps) get(k + kAhead);
      if (k < kValues) {
        acc[k % ND] = mfma32(ring[k & 7], as_h8(w[k / ND]), acc[k % ND]);
      } else {
        const int i = k & 1, f = (k - kValues) >> 1;
        if (f == 0) {
#pragma unroll
          for (int e = 0; e < 16; ++e) s[i][e] = 0.0f;
        }
        s[i] = mfma32(ring[k & 7], q[f], s[i]);
      }
      side(k);
    }
    mfma_drain();
  };
  // Vector half: the weights of the scores.
  TileMeta meta[4];
  const auto weigh = [&](int i_tile) {
    const int pos = u.kv_begin + i_tile * kTileKeys;
    float g[4], lv[4], iv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = meta[i][0] * rowf, lv[i] = meta[i][1], iv[i] = meta[i][2];
    if (__builtin_expect_with_probability(pos + kTileKeys > plain || bad_seen != 0, 0, 0.99)) {
      // some rows do not see all of the tile's keys: a hidden key's score is
      // -inf, and where a lane sees none of 8 keys their block's scales, which
      // may be anything, do not count
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t see = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int n = min(max(limit - pos - 16 * i - 8 * j - 4 * half, 0), 4);
          see |= ((1u << n) - 1u) << (4 * j);
        }
        see = __float_as_int(meta[i][3]) != 0 ? 0 : see;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[i >> 1][8 * (i & 1) + e] = (see >> e) & 1 ? s[i >> 1][8 * (i & 1) + e] : -INFINITY;
        g[i] = see == 0 ? 1.0f : g[i] < 1.1754944e-38f ? 1.1754944e-38f : g[i];  // (-inf times zero is no -inf)
        lv[i] = see == 0 ? kLowest : lv[i];
        iv[i] = see == 0 ? 0.0f : iv[i];
      }
    }
    float dl, dx;
    const auto weights = [&]() {
      dl = dx = 0.0f;
      float most_sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = lv[i] - m;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = exp2_fast(__builtin_fmaf(s[i >> 1][8 * (i & 1) + e], g[i], c));
        w[i] = uint4{pack_f16(p[0], p[1]), pack_f16(p[2], p[3]), pack_f16(p[4], p[5]), pack_f16(p[6], p[7])};
        const half2_t one = {(_Float16)1.0f, (_Float16)1.0f};
        float sum = __builtin_amdgcn_fdot2(as_half2(w[i].x), one, 0.0f, false);
        sum = __builtin_amdgcn_fdot2(as_half2(w[i].y), one, sum, false);
        sum = __builtin_amdgcn_fdot2(as_half2(w[i].z), one, sum, false);
        sum = __builtin_amdgcn_fdot2(as_half2(w[i].w), one, sum, false);
        most_sum = i == 0 ? sum : fmaxf(most_sum, sum);
        dl = __builtin_fmaf(sum, iv[i], dl);
        if constexpr (kLse) dx = __builtin_fmaf(((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])), iv[i], dx);
      }
      return most_sum;
    };
    const float sum = weights();
    if (__builtin_expect_with_probability(__any(sum > sum_limit), 0, 0.999)) {
      float top = kLowest;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fmaf(max8(s[i >> 1], 8 * (i & 1)), g[i], lv[i]));
      top = reference_of(fmaxf(top, __shfl_xor(top, 32, kWave)));
      top = fmaxf(m, top);  // (never down: other rows may have asked)
      const float scale = exp2_fast(m - top);
      m = top;
      sum_limit = is_far(m) ? -1.0f : kSumLimit;
      l *= scale, x *= scale;
#pragma unroll
      for (int n = 0; n < ND; ++n) acc[n] *= scale;
      if (__builtin_expect_with_probability(__any(is_far(m)), 0, 0.999)) {  // the scores become their weights' exponents
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[i >> 1][8 * (i & 1) + e] = far_exponent(s[i >> 1][8 * (i & 1) + e], g[i], lv[i], m);
          g[i] = 1.0f, lv[i] = m;
        }
      }
      (void)weights();
    }
    if (__builtin_expect_with_probability(uneven != 0, 0, 0.99)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = lv[i] - m;
        float rounded = 0.0f, whole = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = exp2_fast(__builtin_fmaf(s[i >> 1][8 * (i & 1) + e], g[i], c));
          whole += p, rounded += (float)(_Float16)p;
        }
        if (rounded < kSmallSum) dl = __builtin_fmaf(whole - rounded, iv[i], dl);
      }
    }
    l += dl;
    if constexpr (kLse) x += dx;
  };

  // Steps.  A tile takes two, matrix and vector half; the first also decodes
  // this wave's codes of another tile, in the shadow of the products.  With 8
  // waves the upper four are one step behind, so that on every SIMD one wave has
  // the matrix cores while the other has the vector unit.  Steps of the lower
  // waves (the upper's are one later):
  //   2 i      values of V(i - 1), scores of K(i); K(i + 1) written; V(i) written (by the upper, in 2 i + 1)
  //   2 i + 1  weights of tile i
  // K(i + 1) takes the place of K(i - 1), last read in step 2 i - 1, and V(i)
  // that of V(i - 2), last read in step 2 i - 1.  The tile's scales are written
  // in the vector half before, four tiles' in turn.
  if (tiles > 0) {
    char* const buf0 = lds;
    char* const buf1 = lds + kTileBytes<D>;
    // before the first step: K(0), its scales, and no values for no weights
    if (!upper) {
#pragma unroll
      for (int t = 0; t < 8; ++t) decode(0, 0, buf0, t);
    }
    store_meta(0);
    for (int i = tid; i < kVBytes / 16; i += NW * kWave) reinterpret_cast<uint4*>(buf1 + kKBytes)[i] = uint4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = uint4{0, 0, 0, 0};
    turn_pages(0, 2);
    if (!upper) fetch(0, 1);
    __syncthreads();
    if (upper) __syncthreads();
    for (int i = 0; i < tiles; ++i) {
      char* const cur = i & 1 ? buf1 : buf0;
      char* const other = i & 1 ? buf0 : buf1;
      // K(i + 1) or V(i) decoded and the next codes fetched, the next tile's
      // scales written, this one's read
      constexpr int kTasks = kRoles * 9 + 2;
      __builtin_amdgcn_s_setprio(1);  // the products go first: the other wave's vector work fills what they leave
      matrix(other, cur, std::true_type{}, [&](int k) {
#pragma unroll
        for (int t = k * kTasks / kAll; t < (k + 1) * kTasks / kAll; ++t) {
          if (t == kTasks - 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) meta[j] = metas[(i & 3) * 4 + j];
          } else if (t == kTasks - 2) {
            store_meta(i + 1);
          } else {
            const int o = t / 9, part_t = t % 9;
            const bool v = kRoles == 2 ? o == 1 : upper;
            if (part_t < 8) decode(o, v ? i : i + 1, v ? cur : other, part_t);
            else fetch(o, v ? i + 1 : i + 2);
          }
        }
      });
      __builtin_amdgcn_s_setprio(0);
      __syncthreads();
      weigh(i);
      turn_pages(i + 1, i + 3);
      if (NW == 8) __syncthreads();
    }
    matrix((tiles - 1) & 1 ? buf1 : buf0, nullptr, std::false_type{}, [](int) {});
    if (NW == 8 && !upper) __syncthreads();
  }
  if (bad_seen != 0 && lane == 0) atomicOr(a.status, NSMLP_STATUS_BLOCK_UNAVAILABLE);

  // a lane's results: D / 32 runs of 16 dims, in pieces of 4
  const auto dim_of = [&](int g) { return (g >> 1) * 64 + (g & 1) * 32 + 16 * half; };
  const auto piece = [&](int g, int i, float f) {
    if constexpr (D == 128) return float4_t{acc[0][4 * g + i], acc[1][4 * g + i], acc[2][4 * g + i], acc[3][4 * g + i]} * f;
    else return float4_t{acc[0][4 * g + i], acc[0][8 + 4 * g + i], acc[1][4 * g + i], acc[1][8 + 4 * g + i]} * f;
  };
  l += __shfl_xor(l, 32, kWave), x += __shfl_xor(x, 32, kWave);
  if (in) {
    if (u.part >= 0) {
      const long long at = ((long long)u.part * a.c.heads + h) * kRows + r;
#pragma unroll
      for (int g = 0; g < D / 32; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<float4_t*>(a.acc_b + at * D + dim_of(g) + 4 * i) = piece(g, i, 1.0f);
      if (half == 0) *reinterpret_cast<float4_t*>(a.ml_b + 4 * at) = float4_t{m, l, x, 0.0f};
    } else {
      const long long at = (long long)(q0 + tok) * a.c.heads * a.group + h * a.group + row % a.group;
      const float inv = inverse_of(l);
#pragma unroll
      for (int g = 0; g < D / 32; ++g) {
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4_t p = piece(g, i, inv);
          o[2 * i] = to_out<kBf16>(p[0]) | (uint32_t)to_out<kBf16>(p[1]) << 16;
          o[2 * i + 1] = to_out<kBf16>(p[2]) | (uint32_t)to_out<kBf16>(p[3]) << 16;
        }
        uint4* to = reinterpret_cast<uint4*>(a.out + at * D + dim_of(g));
        to[0] = uint4{o[0], o[1], o[2], o[3]};
        to[1] = uint4{o[4], o[5], o[6], o[7]};
      }
      if (kLse && half == 0) a.lse[at] = lse_of(m, x);
    }
  }
}

// Both lists in one launch: list b's units first, the longest work of a step.
template <int D, int kFmt, bool kBf16, int NW, bool kLse>
__global__ void __launch_bounds__(NW* kWave, 2) k_attn_both(KvAttnArgs a, int blocks_b) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  kernarg_warm<sizeof(KvAttnArgs)>();
  const int block = blockIdx.x;
  if (block < blocks_b) {
    const int items = min(a.sched[2], a.s.max_units_b) * a.c.heads;
    const KvUnit* units = reinterpret_cast<const KvUnit*>(a.sched + a.s.off_units_b);
    for (int item = block; item < items; item += blocks_b) {
      tile_unit<D, kFmt, kBf16, NW, kLse>(a, load_unit(units + item / a.c.heads), item % a.c.heads, lds);
      __syncthreads();
    }
  } else {
    stream_share<D, kFmt, kBf16, NW>(a, block - blocks_b, *reinterpret_cast<StreamLds<D, NW>*>(lds));
  }
}

// ------------------------------------------------------------------ join --
// Rows of list b whose keys were shared out: weights 2^(m_p - m), eight parts'
// results in flight at a time.  Where there are many rows a wave has one;
// up to 1024 (four per CU) a workgroup has one, every wave takes a quarter of the
// parts, and their sums meet in LDS.  Whole calls, a wave per row against a
// workgroup: 12 tokens of 24 heads over 15692 keys 17.8 us, 16.0; 6 of 12 heads
// over 102424 keys 52.5, 40.8.  With the bound at 4096: 32 tokens of 64 heads over
// 10000 keys (2048 rows) 36.9 us, 40.4; 64 of 32 heads over 40000 59.7, 63.0.
template <int E>
struct JoinSum {
  float m, l, x, o[E];
};

template <int E>
__device__ __forceinline__ JoinSum<E> join_parts(const KvAttnArgs& a, long long first, long long step, int begin, int end, int lane) {
  JoinSum<E> s = {kLowest, 0.0f, 0.0f, {}};
  for (int base = begin; base < end; base += 8) {
    float4_t ml[8];
    float y[8][E];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const long long at = first + min(base + p, end - 1) * step;  // (the last again: no branch between the reads)
      ml[p] = *reinterpret_cast<const float4_t*>(a.ml_b + 4 * at);
#pragma unroll
      for (int e = 0; e < E; ++e) y[p][e] = a.acc_b[(at * kWave + lane) * E + e];
    }
    float top = s.m;
#pragma unroll
    for (int p = 0; p < 8; ++p) top = fmaxf(top, ml[p][0]);
    const float old = exp2_fast(s.m - top);
    s.m = top, s.l *= old, s.x *= old;
#pragma unroll
    for (int e = 0; e < E; ++e) s.o[e] *= old;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const float w = exp2_fast(ml[p][0] - s.m);
      if (base + p < end) {
        s.l += ml[p][1] * w, s.x += ml[p][2] * w;
#pragma unroll
        for (int e = 0; e < E; ++e) s.o[e] += y[p][e] * w;
      }
    }
  }
  return s;
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(256) k_attn_join(KvAttnArgs a) {
  kernarg_warm<sizeof(KvAttnArgs)>();
  constexpr int E = D / kWave;
  __shared__ float part_o[4][D], part_m[4][3];
  const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6), rows_b = a.s.rows_b, rows_j = a.s.join_rows;
  const KvSplit* splits = reinterpret_cast<const KvSplit*>(a.sched + a.s.off_splits_b);
  const int tiles = min(a.sched[3], a.s.max_splits_b), items = tiles * a.c.heads * rows_j;
  const bool wide = items <= 1024;
  const int at_once = wide ? (int)gridDim.x : (int)gridDim.x * 4;
  for (int item = wide ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave; item < items; item += at_once) {
    const int r = item % rows_j, h = item / rows_j % a.c.heads;
    const KvSplit sp = splits[item / rows_j / a.c.heads];
    const int q0 = a.q_start[sp.req], rows = (a.q_start[sp.req + 1] - q0) * a.group;
    const int full = sp.row + r, tok = q0 + full / a.group;
    if (full >= rows || !in_step(a, tok)) continue;  // (the same for all waves of a wide row)
    const long long first = ((long long)sp.first * a.c.heads + h) * rows_b + r, step = (long long)a.c.heads * rows_b;
    const int each = wide ? (sp.parts + 3) >> 2 : sp.parts, begin = wide ? min(wave * each, sp.parts) : 0;
    JoinSum<E> s = join_parts<E>(a, first, step, begin, min(begin + each, sp.parts), lane);
    if (wide) {
      __syncthreads();  // (the row before has been read)
      if (lane == 0) part_m[wave][0] = s.m, part_m[wave][1] = s.l, part_m[wave][2] = s.x;
#pragma unroll
      for (int e = 0; e < E; ++e) part_o[wave][lane * E + e] = s.o[e];
      __syncthreads();
      if (wave != 0) continue;
      float top = kLowest;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, part_m[w][0]);
      s = {top, 0.0f, 0.0f, {}};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = exp2_fast(part_m[w][0] - top);
        s.l += part_m[w][1] * f, s.x += part_m[w][2] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) s.o[e] += part_o[w][lane * E + e] * f;
      }
    }
    const float inv = inverse_of(s.l);
    const long long at = (long long)tok * a.c.heads * a.group + h * a.group + full % a.group;
    if constexpr (E == 2)
      *reinterpret_cast<uint32_t*>(a.out + at * D + lane * 2) =
          to_out<kBf16>(s.o[0] * inv) | (uint32_t)to_out<kBf16>(s.o[1] * inv) << 16;
    else
      a.out[at * D + lane] = to_out<kBf16>(s.o[0] * inv);
    if (a.lse != nullptr && lane == 0) a.lse[at] = lse_of(s.m, s.x);
  }
}

template <int D, int kFmt, bool kBf16, int NW, bool kLse>
void launch_both(const KvAttnArgs& a, int stream_blocks, hipStream_t s) {
  constexpr int kStream = (int)sizeof(StreamLds<D, NW>), kLds = kStream > kTileLds<D> ? kStream : kTileLds<D>;
  static std::once_flag once;
  std::call_once(once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_attn_both<D, kFmt, kBf16, NW, kLse>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  });
  const int blocks_b = (int)min((long long)a.s.max_units_b * a.c.heads, 65536LL);
  k_attn_both<D, kFmt, kBf16, NW, kLse><<<dim3(blocks_b + stream_blocks), dim3(NW * kWave), kLds, s>>>(a, blocks_b);
}

template <int D, int kFmt, bool kBf16>
void attention_typed(const KvAttnArgs& a, hipStream_t s) {
  const int stream_blocks = (a.s.shares + 7) / 8 * 8 * a.c.heads;
  if (!a.s.list_b) {
    k_attn_stream<D, kFmt, kBf16><<<dim3(stream_blocks), dim3(4 * kWave), 0, s>>>(a);
    return;
  }
  const bool lse = a.lse != nullptr;
  if (a.s.rows_b == 256) lse ? launch_both<D, kFmt, kBf16, 8, true>(a, stream_blocks, s) : launch_both<D, kFmt, kBf16, 8, false>(a, stream_blocks, s);
  else lse ? launch_both<D, kFmt, kBf16, 4, true>(a, stream_blocks, s) : launch_both<D, kFmt, kBf16, 4, false>(a, stream_blocks, s);
  if (a.s.max_splits_b > 0) {
    const long long waves = (long long)a.s.max_splits_b * a.c.heads * a.s.join_rows;
    k_attn_join<D, kBf16><<<dim3((unsigned)min((waves + 3) / 4, 1024LL)), dim3(256), 0, s>>>(a);
  }
}

}  // namespace

size_t kv_attn_partial_floats(const KvSchedule& s, int kv_heads, int D, size_t (&off)[4]) {
  size_t at = 0;
  const size_t ra = (size_t)s.max_parts_a * kv_heads * kKvRowsA, rb = (size_t)s.max_parts_b * kv_heads * s.rows_b;
  off[0] = at, at += ra * D;
  off[1] = at, at += ra * 2;
  off[2] = at, at += rb * D;
  off[3] = at, at += rb * 4;
  return at;
}

void launch_kv_attention(const KvAttnArgs& a, bool bf16, hipStream_t s) {
  NSMLP_KV_BY_TYPE(attention_typed, a, bf16, s);
}

}  // namespace nsmlp
