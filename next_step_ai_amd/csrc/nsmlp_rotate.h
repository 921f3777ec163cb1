// Rotary position encoding of rows on their way into the K/V cache, and of the
// query rows next to them.
//
// A pair (a, b) of a row's dims becomes (a c - b s, b c + a s), c and s the fp32
// cos and sin of its angle from the table.  Products of a 16-bit value and an
// fp32 one are exact in 64 bits, so the fused sum below is the exact one rounded
// once; then it is rounded to fp32 and to the rows' type.  The result does not
// depend on who computes it, which is what lets codes be compared bit for bit
// with those of rows rotated beforehand.  (64-bit operations run at half the
// fp32 rate here and stay hidden behind the rows' way through memory.)
#pragma once

#include "nsmlp_kv.h"

namespace nsmlp {

template <bool kBf16>
__device__ __forceinline__ float in_value(uint32_t h) {
  if constexpr (kBf16) return __uint_as_float(h << 16);
  else return h2f((uint16_t)h);
}
template <bool kBf16>
__device__ __forceinline__ float in_lo(uint32_t w) { return in_value<kBf16>(w & 0xFFFFu); }
template <bool kBf16>
__device__ __forceinline__ float in_hi(uint32_t w) {
  if constexpr (kBf16) return __uint_as_float(w & 0xFFFF0000u);
  else return in_value<kBf16>(w >> 16);
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (kBf16) return __builtin_bit_cast(uint16_t, (__bf16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16;
  else return f2h(a) | (uint32_t)f2h(b) << 16;
}

// What N neighbouring dims from d0 on are multiplied by: x c + partner s.  NaN
// for a position outside the table.
template <int N>
struct Angles {
  float c[N], s[N];
};
template <int D, int N>
__device__ __forceinline__ Angles<N> angles_of(const KvRotateArgs& r, int pos, int d0) {
  Angles<N> o;
  const bool in = (unsigned)pos < (unsigned)r.reach;
  const float* row = r.table + (long long)(in ? pos : 0) * D;
  if (r.interleaved) {
    const float4* p = reinterpret_cast<const float4*>(row + d0);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = p[i];
      o.c[4 * i] = o.c[4 * i + 1] = v.x, o.c[4 * i + 2] = o.c[4 * i + 3] = v.z;
      o.s[4 * i] = -v.y, o.s[4 * i + 1] = v.y, o.s[4 * i + 2] = -v.w, o.s[4 * i + 3] = v.w;
    }
  } else {
    const bool upper = d0 >= D / 2;
    const float4* p = reinterpret_cast<const float4*>(row + 2 * (upper ? d0 - D / 2 : d0));
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float4 v = p[i];
      o.c[2 * i] = v.x, o.c[2 * i + 1] = v.z;
      o.s[2 * i] = upper ? v.y : -v.y, o.s[2 * i + 1] = upper ? v.w : -v.w;
    }
  }
  if (!in) {
#pragma unroll
    for (int i = 0; i < N; ++i) o.c[i] = o.s[i] = __uint_as_float(0x7FC00000u);
  }
  return o;
}

__device__ __forceinline__ float rotate1(float x, float y, float c, float s) {
  float f = (float)__builtin_fma((double)x, (double)c, (double)y * (double)s);
  asm("" : "+v"(f));  // both roundings: the compiler would make one of the two, from 64 bits to the rows' type
  return f;
}

// N / 2 dwords of a row whose partners D / 2 dims away are in `other`.
template <int N, bool kBf16>
__device__ __forceinline__ void rotate(uint32_t (&x)[N / 2], const uint32_t (&other)[N / 2], const Angles<N>& a, bool interleaved) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const uint32_t y = interleaved ? x[i] >> 16 | x[i] << 16 : other[i];
    x[i] = pack_out<kBf16>(rotate1(in_lo<kBf16>(x[i]), in_lo<kBf16>(y), a.c[2 * i], a.s[2 * i]),
                           rotate1(in_hi<kBf16>(x[i]), in_hi<kBf16>(y), a.c[2 * i + 1], a.s[2 * i + 1]));
  }
}

// A lane's D/16 dims of a row that 16 lanes hold: D/32 dwords.
template <int D>
struct RowPart {
  uint32_t w[D / 32];
};
template <int D>
__device__ __forceinline__ RowPart<D> load_part(const uint16_t* p) {
  RowPart<D> o;
  if constexpr (D == 128) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    o.w[0] = v.x, o.w[1] = v.y, o.w[2] = v.z, o.w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    o.w[0] = v.x, o.w[1] = v.y;
  }
  return o;
}
template <int D>
__device__ __forceinline__ void store_part(uint16_t* p, const RowPart<D>& v) {
  if constexpr (D == 128) *reinterpret_cast<uint4*>(p) = uint4{v.w[0], v.w[1], v.w[2], v.w[3]};
  else *reinterpret_cast<uint2*>(p) = uint2{v.w[0], v.w[1]};
}
// The partners of all lanes are 8 lanes on, in the row of 16.  (All lanes active.)
template <int D, bool kBf16>
__device__ __forceinline__ void rotate_part(RowPart<D>& x, const Angles<D / 16>& a, bool interleaved) {
  uint32_t other[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) other[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x.w[i], 0x128, 0xf, 0xf, true);  // row_ror:8
  rotate<D / 16, kBf16>(x.w, other, a, interleaved);
}

// Query rows: 16 lanes turn kQueryHeads heads of a token under one set of
// angles (8 bytes a pair: a token's are as much as two heads' rows).  `unit` counts
// tokens times groups of heads.  HBM bounds it: an append of 12071 tokens takes 20
// us without and 49 us with 32 heads of 128 (198 MB in and out).
constexpr int kQueryHeads = 4;
__host__ __device__ __forceinline__ long long query_units(const KvRotateArgs& r, int n) {
  return (long long)n * ((r.q_heads + kQueryHeads - 1) / kQueryHeads);
}
template <int D, bool kBf16>
__device__ __forceinline__ void rotate_queries(const KvRotateArgs& r, int n, long long unit, int lane) {
  constexpr int E = D / 16;
  const int groups = (r.q_heads + kQueryHeads - 1) / kQueryHeads;
  const long long t_of = unit / groups;
  const int t = (int)min(t_of, (long long)n - 1), h0 = (int)(unit % groups) * kQueryHeads, d0 = (lane & 15) * E;
  const int pos = t_of < n ? r.positions[t] : -1;
  const uint16_t* from = r.q + (long long)t * r.q_row + d0;
  RowPart<D> x[kQueryHeads];
#pragma unroll
  for (int i = 0; i < kQueryHeads; ++i) x[i] = load_part<D>(from + (long long)min(h0 + i, r.q_heads - 1) * r.q_head);
  const Angles<E> a = angles_of<D, E>(r, pos, d0);
#pragma unroll
  for (int i = 0; i < kQueryHeads; ++i) rotate_part<D, kBf16>(x[i], a, r.interleaved);
  if (pos < 0) return;
  uint16_t* to = r.q_out + (long long)t * r.out_row + d0;
#pragma unroll
  for (int i = 0; i < kQueryHeads; ++i)
    if (h0 + i < r.q_heads) store_part<D>(to + (long long)(h0 + i) * r.out_head, x[i]);
}

}  // namespace nsmlp
