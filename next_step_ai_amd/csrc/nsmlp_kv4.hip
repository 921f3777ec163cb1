// Append and read of the 4-bit K/V cache (layout: nsmlp_kv.h).
//
// A value x of 32 neighbouring dims with largest magnitude a becomes the e2m1
// code nearest to x / 2^e (ties to the even one), e the least exponent with a <=
// 6 2^e between -23 and 13.  The conversion instructions take the 16-bit values
// and the scale as they are and round so; past the largest code they saturate.
// The scale is a token's own, so no stored token is read again.
#include <type_traits>

#include "nsmlp_rotate.h"

namespace nsmlp {

namespace {

typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));

// ---------------------------------------------------------------- append --
// 16 lanes per (token, head): each holds D/16 neighbouring dims of K and of V,
// which is a piece of either tile, and 2 (4) or 4 (8) lanes meet over DPP for the
// largest magnitude of 32 dims.  A wave has four neighbouring tokens of a head, whose
// bytes stand next to each other in the tiles.  Query rows follow in workgroups
// of their own.
//
// What bounds it: the rows' way from HBM, and the queries' way in and out.  12071
// tokens of 8 heads of 128 (49 MB in, 13 MB out) 14 us, 4.4 TB/s; K rotated on
// the way 20.9 us (6 MB of angles, and position and angles one after the other before a
// row can be stored; a kernel without the query branch, whose 40 registers leave room for
// all eight waves a SIMD where 109 leave it for four, 20.2); with 32 heads of queries (198
// MB more) 50 us, 5.2 TB/s.  Few tokens take one chain of slot, rows,
// positions, angles: 1 token 2.8 us, 64 tokens with their queries 3.5.
constexpr int kAppend4Threads = 256;

// larger of v and what the other lanes of 4 (D = 128) or 8 hold
template <int D>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));  // quad_perm 2 3 0 1
  if constexpr (D == 64) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // row_half_mirror
  return v;
}

// Scale byte of 32 dims whose largest magnitude is `top` (bits of a finite value).
template <bool kBf16>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  // with a = m 2^E: E - 2 where m <= 1.5, else E - 1 (a subnormal fp32 value is below the least anyway)
  const int e = (int)((__float_as_uint(in_value<kBf16>(top)) + 0x3FFFFFu) >> 23) - 127 - 2;
  return (uint32_t)(min(max(e, kKv4Least), kKv4Most) + 127);
}

// Codes of 8 values, 4 dwords of 16-bit pairs (of 4 values, 2 dwords: in the low half).
template <int W, bool kBf16>
__device__ __forceinline__ uint32_t encode4(const uint32_t (&x)[W], uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  uint32_t o = 0;
  if constexpr (kBf16) {
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf2_t, x[0]), s, 0);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf2_t, x[1]), s, 1);
    if constexpr (W == 4) {
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf2_t, x[2]), s, 2);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf2_t, x[3]), s, 3);
    }
  } else {
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, as_half2(x[0]), s, 0);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, as_half2(x[1]), s, 1);
    if constexpr (W == 4) {
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, as_half2(x[2]), s, 2);
      o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o, as_half2(x[3]), s, 3);
    }
  }
  return o;
}

template <int D>
__device__ __forceinline__ void put_codes(uint8_t* p, uint32_t codes) {
  if constexpr (D == 128) *reinterpret_cast<uint32_t*>(p) = codes;
  else *reinterpret_cast<uint16_t*>(p) = (uint16_t)codes;
}

template <int D, bool kBf16, bool kRotate>
__global__ void __launch_bounds__(kAppend4Threads) k_kv_append4(KvAppendArgs a) {
  kernarg_warm<sizeof(KvAppendArgs)>();
  constexpr int E = D / 16;
  const int lane = threadIdx.x & (kWave - 1), r = lane & 15;
  if (kRotate && blockIdx.x >= a.rot.first) {
    rotate_queries<D, kBf16>(a.rot, a.n, (long long)(blockIdx.x - a.rot.first) * (kAppend4Threads / 16) + (threadIdx.x >> 4), lane);
    return;
  }
  const unsigned unit = blockIdx.x * (unsigned)(kAppend4Threads / 16) + (threadIdx.x >> 4);
  const unsigned th = unit >> 2;
  const int h = (int)(th % (unsigned)a.c.heads);
  const long long t = (long long)(th / (unsigned)a.c.heads) * 4 + (unit & 3);
  const bool in = t < a.n;
  const long long ta = in ? t : 0;
  const long long slot = in ? a.slots[ta] : -1;
  RowPart<D> k = load_part<D>(a.k + ta * a.k_row + (long long)h * a.k_head + r * E);
  const RowPart<D> v = load_part<D>(a.v + ta * a.v_row + (long long)h * a.v_head + r * E);
  if constexpr (kRotate) rotate_part<D, kBf16>(k, angles_of<D, E>(a.rot, a.rot.positions[ta], r * E), a.rot.interleaved);
  uint32_t top_k = 0, top_v = 0;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    top_k = max(top_k, max(k.w[i] & 0x7FFFu, (k.w[i] >> 16) & 0x7FFFu));
    top_v = max(top_v, max(v.w[i] & 0x7FFFu, (v.w[i] >> 16) & 0x7FFFu));
  }
  top_k = group_max<D>(top_k), top_v = group_max<D>(top_v);
  // a value that is not finite anywhere in the token's K or V
  const unsigned long long odd = __ballot(max(top_k, top_v) >= (kBf16 ? 0x7F80u : 0x7C00u));
  const bool bad = ((odd >> (lane & 48)) & 0xFFFFull) != 0;
  const uint32_t byte_k = bad ? kKv4Bad : scale_byte<kBf16>(top_k), byte_v = bad ? 127 + kKv4Least : scale_byte<kBf16>(top_v);
  const uint32_t codes_k = bad ? 0 : encode4<D / 32, kBf16>(k.w, byte_k), codes_v = bad ? 0 : encode4<D / 32, kBf16>(v.w, byte_v);
  if (slot < 0 || slot >= (long long)a.c.num_blocks * a.c.B) return;
  const int B = a.c.B, off = (int)(slot & (B - 1));
  uint8_t* to = a.c.data + ((slot >> a.c.b_shift) * a.c.heads + h) * kv_block_bytes<NSMLP_KV_E2M1>(B, D);
  put_codes<D>(to + kv4_k_off(D, off, r), codes_k);
  put_codes<D>(to + B * D / 2 + kv4_v_off(D, off, r), codes_v);
  constexpr int kLanes = 32 / E;  // of a scale
  if (r % kLanes == 0) {
    to[B * D + kv4_ks_off(D, off, r / kLanes)] = (uint8_t)byte_k;
    to[B * D + B * D / 32 + kv4_vs_off(D, off, r / kLanes)] = (uint8_t)byte_v;
  }
}

// ------------------------------------------------------------------ read --
// 16 lanes per (slot, head), D/16 dims of K and V each; every value is a number
// of either type.  HBM bounds it, most of it what is written: 12071 slots of 8
// heads of 128 (13 MB in, 49 MB out) 15.8 us, 3.9 TB/s; 1 slot 2.5 us.
template <int D, bool kBf16>
__device__ __forceinline__ RowPart<D> decode4(uint32_t codes, uint32_t byte) {
  const float s = __uint_as_float(byte << 23);
  RowPart<D> o;
  const auto pair = [&](auto at) {
    constexpr int i = decltype(at)::value;
    if constexpr (kBf16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, s, i));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, s, i));
  };
  o.w[0] = pair(std::integral_constant<int, 0>{});
  o.w[1] = pair(std::integral_constant<int, 1>{});
  if constexpr (D == 128) {
    o.w[2] = pair(std::integral_constant<int, 2>{});
    o.w[3] = pair(std::integral_constant<int, 3>{});
  }
  return o;
}

template <int D>
__device__ __forceinline__ uint32_t get_codes(const uint8_t* p) {
  if constexpr (D == 128) return *reinterpret_cast<const uint32_t*>(p);
  else return *reinterpret_cast<const uint16_t*>(p);
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(256) k_kv_read4(KvReadArgs a) {
  kernarg_warm<sizeof(KvReadArgs)>();
  constexpr int E = D / 16, kLanes = 32 / E;
  const unsigned unit = blockIdx.x * 16u + (threadIdx.x >> 4);
  const int r = threadIdx.x & 15, h = (int)(unit % (unsigned)a.c.heads), t = (int)(unit / (unsigned)a.c.heads);
  if (t >= a.n) return;
  const long long slot = a.slots[t];
  RowPart<D> k = {}, v = {};
  if (slot >= 0 && slot < (long long)a.c.num_blocks * a.c.B) {
    const int B = a.c.B, off = (int)(slot & (B - 1));
    const uint8_t* from = a.c.data + ((slot >> a.c.b_shift) * a.c.heads + h) * kv_block_bytes<NSMLP_KV_E2M1>(B, D);
    const uint32_t ck = get_codes<D>(from + kv4_k_off(D, off, r)), cv = get_codes<D>(from + B * D / 2 + kv4_v_off(D, off, r));
    const uint32_t sk = from[B * D + kv4_ks_off(D, off, r / kLanes)], sv = from[B * D + B * D / 32 + kv4_vs_off(D, off, r / kLanes)];
    k = decode4<D, kBf16>(ck, sk);
    v = decode4<D, kBf16>(cv, sk == kKv4Bad ? kKv4Bad : sv);
    if (sk == kKv4Bad) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) k.w[i] = v.w[i] = kBf16 ? 0x7FC07FC0u : 0x7E007E00u;
    }
  }
  const long long o = ((long long)t * a.c.heads + h) * D + r * E;
  store_part<D>(a.k + o, k);
  store_part<D>(a.v + o, v);
}

template <int D, bool kBf16>
void append4_typed(KvAppendArgs a, hipStream_t s) {
  constexpr int kUnits = kAppend4Threads / 16;
  const long long units = (long long)((a.n + 3) / 4) * 4 * a.c.heads;
  a.rot.first = (unsigned)((units + kUnits - 1) / kUnits);
  const long long queries = a.rot.q != nullptr ? query_units(a.rot, a.n) : 0;
  const dim3 grid(a.rot.first + (unsigned)((queries + kUnits - 1) / kUnits)), block(kAppend4Threads);
  if (a.rot.table != nullptr) k_kv_append4<D, kBf16, true><<<grid, block, 0, s>>>(a);
  else k_kv_append4<D, kBf16, false><<<grid, block, 0, s>>>(a);
}

template <int D, bool kBf16>
void read4_typed(const KvReadArgs& a, hipStream_t s) {
  const long long units = (long long)a.n * a.c.heads;
  k_kv_read4<D, kBf16><<<dim3((unsigned)((units + 15) / 16)), dim3(256), 0, s>>>(a);
}

}  // namespace

void launch_kv_append4(const KvAppendArgs& a, bool bf16, hipStream_t s) {
  if (a.c.D == 128) bf16 ? append4_typed<128, true>(a, s) : append4_typed<128, false>(a, s);
  else bf16 ? append4_typed<64, true>(a, s) : append4_typed<64, false>(a, s);
}
void launch_kv_read4(const KvReadArgs& a, bool bf16, hipStream_t s) {
  if (a.c.D == 128) bf16 ? read4_typed<128, true>(a, s) : read4_typed<128, false>(a, s);
  else bf16 ? read4_typed<64, true>(a, s) : read4_typed<64, false>(a, s);
}

}  // namespace nsmlp
