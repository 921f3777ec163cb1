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
// exactly.  m follows the running maximum lazily: it moves only where a tile
// exceeds it by more than 2^8, so most tiles neither rescale acc nor exchange
// maxima between lanes; a weight is then at most 2^8, far inside fp16.
// acc, l, m and the scores are fp32; a weight is rounded to fp16 once, as the
// products' operand (relative 2^-12, averaged over the keys).
#include <mutex>
#include <type_traits>

#include "nsmlp_kv.h"

namespace nsmlp {

namespace {

constexpr float kLowest = -3.402823466e38f;
constexpr float kLazy = 8.0f;

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

// Pages of a range of keys, held one per lane: 64 pages from page `first`.
struct Pages {
  int id;          // block id (0 where the entry is not a block)
  float ks, lv, iv;  // K scale, log2 and reciprocal of the V scale
  unsigned long long bad;
  int first;
};

__device__ __forceinline__ Pages load_pages(const KvAttnArgs& a, int req, int h, int first, int last, int lane) {
  Pages p;
  p.first = first;
  const int pg = min(min(first + lane, last), a.max_blocks - 1);
  const int id = a.table[(long long)req * a.max_blocks + pg];
  const bool ok = id >= 0 && id < a.c.num_blocks;
  p.id = ok ? id : 0;
  const float2 s = *reinterpret_cast<const float2*>(a.c.scale + ((long long)p.id * a.c.heads + h) * 2);
  const float sv = s.y == 0.0f ? kKvScaleMin : s.y;  // a block that nothing was stored in
  p.bad = __ballot(!ok);
  p.ks = s.x;
  p.lv = log2_fast(sv);
  p.iv = 1.0f / sv;
  return p;
}

__device__ __forceinline__ float lane_of(float v, int i) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i));
}

// ---------------------------------------------------------------- stream --
// Up to 16 NB query rows against a range of keys.  A workgroup is one unit and
// K/V head; its 4 waves share the keys out and their results meet in LDS.
// Products with the keys (or dims) as rows and the queries as columns.
constexpr int kStreamThreads = 256;
constexpr int kStreamWaves = kStreamThreads / kWave;

template <int D, int kFmt>
struct StreamTile {  // 32 keys: two tiles of 16
  uint4 k[2][D / 64], v[2][D / 64];
};

template <int D, int kFmt>
__device__ __forceinline__ void load_tile(StreamTile<D, kFmt>& t, const KvAttnArgs& a, const Pages& p, int h, int pos,
                                          int last, int lane) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int at = pos + 16 * s;
    const int pg = min(at >> a.c.b_shift, last);
    const int id = __builtin_amdgcn_readlane(p.id, pg - p.first);
    const uint8_t* kb = a.c.data + ((long long)id * a.c.heads + h) * 2 * (a.c.B * D) + ((at & (a.c.B - 1)) >> 4) * (16 * D);
    const uint8_t* vb = kb + a.c.B * D;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      t.k[s][j] = *reinterpret_cast<const uint4*>(kb + j * 1024 + lane * 16);
      t.v[s][j] = *reinterpret_cast<const uint4*>(vb + j * 1024 + lane * 16);
    }
  }
}

template <int D, int kFmt, bool kBf16, int NB>
__global__ void __launch_bounds__(kStreamThreads) k_attn_stream(KvAttnArgs a, const KvUnit* units, const int32_t* n_units,
                                                                int max_units, int rows_of_unit, float* acc_out, float* ml_out) {
  constexpr int NJ = D / 64, KS = D / 32, ND = D / 16, kPad = D + 4;
  __shared__ __attribute__((aligned(16))) float sum_s[kStreamWaves][16][kPad];
  __shared__ float ml_s[kStreamWaves][3][16 * NB];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const bool want_lse = a.lse != nullptr;
  const int items = min(*n_units, max_units) * a.c.heads;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int h = item % a.c.heads;
    const KvUnit u = units[item / a.c.heads];
    const int q0 = a.q_start[u.req], q_len = a.q_start[u.req + 1] - q0, kv_len = a.kv_len[u.req];
    const int rows = min(q_len * a.group - u.row, rows_of_unit);

    // queries: columns of the products, 8 dims per lane and step
    half8_t q[NB][KS];
    float rowf[NB];
    int limit[NB];  // keys that the row sees
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int r = b * 16 + col, row = u.row + r, tok = row / a.group;
      const bool in = r < rows && q0 + tok < a.total;
      limit[b] = in ? kv_len - q_len + tok + 1 : 0x7FFFFFFF;
      const uint16_t* src = a.q + (long long)(q0 + tok) * a.q_row + (long long)(h * a.group + row % a.group) * a.q_head;
      uint4 raw[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s)
        raw[s] = in ? *reinterpret_cast<const uint4*>(src + 64 * (s >> 1) + 16 * grp + 8 * (s & 1)) : uint4{0, 0, 0, 0};
      rowf[b] = a.scale_log2;
      if constexpr (kBf16) {
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = max(top, max(word(raw[s], i) & 0x7FFFu, (word(raw[s], i) >> 16) & 0x7FFFu));
        top = max(top, (uint32_t)__shfl_xor((int)top, 16, kWave));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32, kWave));
        const int e = row_exponent(top);
        rowf[b] *= ldexpf(1.0f, e);
#pragma unroll
        for (int s = 0; s < KS; ++s) q[b][s] = as_h8(bf16_to_f16(raw[s], e));
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) q[b][s] = as_h8(raw[s]);
      }
    }

    // this wave's keys
    const int n = u.kv_end - u.kv_begin;
    const int each = ((n + kStreamWaves - 1) / kStreamWaves + 31) & ~31;
    const int begin = u.kv_begin + wave * each, end = min(begin + each, u.kv_end);
    const int last = max(0, (u.kv_end - 1) >> a.c.b_shift);
    // keys below this need no mask: every row of the unit sees them
    const int plain = kv_len - q_len + u.row / a.group + 1;

    float m[NB], l[NB], x[NB];  // reference, sum of the rounded weights, sum of the weights
    float4_t acc[NB][ND];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      m[b] = kLowest, l[b] = x[b] = 0.0f;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[b][d] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    unsigned long long bad_seen = 0;

    if (begin < end) {
      Pages pages = load_pages(a, u.req, h, begin >> a.c.b_shift, last, lane);
      bad_seen = pages.bad;
      auto use = [&](const StreamTile<D, kFmt>& t, int pos, const Pages& p) {
        float4_t sc[NB][2];
        float f[2], lv[2], iv[2];
        bool bad[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int pg = min((pos + 16 * s) >> a.c.b_shift, last) - p.first;
          f[s] = lane_of(p.ks, pg), lv[s] = lane_of(p.lv, pg), iv[s] = lane_of(p.iv, pg);
          bad[s] = (p.bad >> pg) & 1;
          half8_t kh[KS];
#pragma unroll
          for (int x = 0; x < KS; ++x)
            kh[x] = join4(kv_half4<kFmt>(word(t.k[s][x >> 1], 2 * (x & 1))), kv_half4<kFmt>(word(t.k[s][x >> 1], 2 * (x & 1) + 1)));
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            float4_t c = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < KS; ++x) c = mfma16(kh[x], q[b][x], c);
            sc[b][s] = c;
          }
        }
        const bool masked = pos + 32 > plain || bad[0] || bad[1];
        half8_t w[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float e[2][4], top = kLowest;
          unsigned seen = 0xFF;
          if (masked) {
            seen = 0;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                seen |= (pos + 16 * s + 4 * grp + i < limit[b] && !bad[s]) ? 1u << (4 * s + i) : 0u;
          }
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              e[s][i] = __builtin_fmaf(sc[b][s][i], f[s] * rowf[b], lv[s]);
              if (masked && !((seen >> (4 * s + i)) & 1)) e[s][i] = kLowest;
              top = fmaxf(top, e[s][i]);
            }
          if (__builtin_expect_with_probability(__any(top > m[b] + kLazy), 0, 0.99)) {
            top = fmaxf(top, m[b]);
            top = fmaxf(top, __shfl_xor(top, 16, kWave));
            top = ceilf(fmaxf(top, __shfl_xor(top, 32, kWave)));  // an integer: rescaling is exact
            const float scale = exp2_fast(m[b] - top);
            m[b] = top;
            l[b] *= scale, x[b] *= scale;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[b][d] *= scale;
          }
          float p[2][4];
          uint2 pw[2];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              p[s][i] = exp2_fast(e[s][i] - m[b]);
              if (masked && !((seen >> (4 * s + i)) & 1)) p[s][i] = 0.0f;
            }
            // the sum takes the weights as the products see them, rounded to
            // fp16: where few keys carry the row, their rounding cancels
            pw[s] = uint2{pack_f16(p[s][0], p[s][1]), pack_f16(p[s][2], p[s][3])};
            const half2_t one = {(_Float16)1.0f, (_Float16)1.0f};
            const float sum = __builtin_amdgcn_fdot2(as_half2(pw[s].y), one,
                                                     __builtin_amdgcn_fdot2(as_half2(pw[s].x), one, 0.0f, false), false);
            const bool none = masked && !((seen >> (4 * s)) & 0xF);
            l[b] += none ? 0.0f : sum * iv[s];
            if (want_lse) x[b] += none ? 0.0f : ((p[s][0] + p[s][1]) + (p[s][2] + p[s][3])) * iv[s];
          }
          w[b] = join4(pw[0], pw[1]);
        }
        // codes past the end may be e4m3 NaNs: a zero weight does not hide them
        uint32_t keep[2] = {~0u, ~0u};
        if (kFmt == NSMLP_KV_E4M3 && masked) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const int left = bad[s] ? 0 : kv_len - (pos + 16 * s + 4 * grp);
            keep[s] = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
          }
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const half8_t vh = join4(kv_half4<kFmt>(word(t.v[0][d >> 2], d & 3) & keep[0]),
                                   kv_half4<kFmt>(word(t.v[1][d >> 2], d & 3) & keep[1]));
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b][d] = mfma16(vh, w[b], acc[b][d]);
        }
      };
      StreamTile<D, kFmt> t;
      load_tile(t, a, pages, h, begin, last, lane);
      for (int pos = begin; pos < end; pos += 32) {
        StreamTile<D, kFmt> next = t;
        Pages np = pages;
        if (pos + 32 < end) {
          const int hi = min((pos + 63) >> a.c.b_shift, last);  // the next tile's last page
          if (hi - pages.first >= kWave) {
            np = load_pages(a, u.req, h, (pos + 32) >> a.c.b_shift, last, lane);
            bad_seen |= np.bad;
          }
          load_tile(next, a, np, h, pos + 32, last, lane);
        }
        use(t, pos, pages);
        t = next;
        pages = np;
      }
    }
    if (bad_seen != 0 && lane == 0) atomicOr(a.status, NSMLP_STATUS_BLOCK_UNAVAILABLE);

    // join the waves
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      l[b] += __shfl_xor(l[b], 16, kWave), x[b] += __shfl_xor(x[b], 16, kWave);
      l[b] += __shfl_xor(l[b], 32, kWave), x[b] += __shfl_xor(x[b], 32, kWave);
      if (grp == 0) ml_s[wave][0][b * 16 + col] = m[b], ml_s[wave][1][b * 16 + col] = l[b], ml_s[wave][2][b * 16 + col] = x[b];
    }
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float top = kLowest;
#pragma unroll
      for (int w = 0; w < kStreamWaves; ++w) top = fmaxf(top, ml_s[w][0][b * 16 + col]);
      const float scale = exp2_fast(m[b] - top);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4_t*>(&sum_s[wave][col][64 * j + 16 * grp + 4 * i]) =
              float4_t{acc[b][4 * j][i], acc[b][4 * j + 1][i], acc[b][4 * j + 2][i], acc[b][4 * j + 3][i]} * scale;
      __syncthreads();
      // 16 threads per row, D / 16 dims each
      const int r = tid >> 4, d0 = (tid & 15) * (D / 16), row = b * 16 + r;
      float mr = kLowest, lr = 0.0f, xr = 0.0f;
#pragma unroll
      for (int w = 0; w < kStreamWaves; ++w) mr = fmaxf(mr, ml_s[w][0][row]);
#pragma unroll
      for (int w = 0; w < kStreamWaves; ++w) {
        const float f = exp2_fast(ml_s[w][0][row] - mr);
        lr += ml_s[w][1][row] * f, xr += ml_s[w][2][row] * f;
      }
      float o[D / 16];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        o[d] = sum_s[0][r][d0 + d];
#pragma unroll
        for (int w = 1; w < kStreamWaves; ++w) o[d] += sum_s[w][r][d0 + d];
      }
      if (row < rows) {
        if (u.part >= 0) {
          const long long at = ((long long)u.part * a.c.heads + h) * rows_of_unit + row;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) acc_out[at * D + d0 + d] = o[d];
          if (d0 == 0) *reinterpret_cast<float4_t*>(ml_out + 4 * at) = float4_t{mr, lr, xr, 0.0f};
        } else {
          const int full = u.row + row, tok = q0 + full / a.group, head = h * a.group + full % a.group;
          if (tok < a.total) {
            const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
            const long long at = (long long)tok * a.c.heads * a.group + head;
#pragma unroll
            for (int d = 0; d < D / 16; d += 2)
              *reinterpret_cast<uint32_t*>(a.out + at * D + d0 + d) =
                  to_out<kBf16>(o[d] * inv) | (uint32_t)to_out<kBf16>(o[d + 1] * inv) << 16;
            if (a.lse != nullptr && d0 == 0) a.lse[at] = xr == 0.0f ? -INFINITY : (mr + log2f(xr)) * 0.6931471805599453f;
          }
        }
      }
      __syncthreads();
    }
  }
}

// ----------------------------------------------------------------- tiles --
// Prompts and chunks: NW waves of 32 query rows each against tiles of 64 keys
// that the workgroup decodes to fp16 once, in LDS, as the operands of
// v_mfma_f32_32x32x16_f16 (A rows: keys or dims, B columns: queries):
//   K fragment (32 keys, 16 dims): lane l: key l % 32, dims 16 (2 a + l / 32) + 8 u + 0..7
//   V fragment (32 dims, 16 keys): lane l: keys 4 h + 0..3 and 8 + 4 h + 0..3, h = l / 32
// so that the scores of a query stay in its two lanes, in the order in which
// the second product wants the weights.
//
// A tile's weights are taken under the reference as it stands; their sums, kept
// anyway, tell whether one was too large for it (the first tile, and seldom
// after), and only then is the maximum looked for.  References are integers,
// so that rescaling is exact.
constexpr int kTileKeys = 64;
constexpr float kSumLimit = 4096.0f;  // 16 weights of a lane: none above 2^12, far inside fp16

__device__ __forceinline__ float max16(const float16_t& s, int at) {
  return fmaxf(fmaxf(fmaxf(s[at], s[at + 1]), fmaxf(s[at + 2], s[at + 3])),
               fmaxf(fmaxf(s[at + 4], s[at + 5]), fmaxf(s[at + 6], s[at + 7])));
}

// What the products of a tile need to know of its blocks, per 16 keys.
struct TileMeta {
  float4_t ks, lv, iv;
  int bad[4];
};

template <int D, int kFmt, bool kBf16, int NW, bool kLse>
__global__ void __launch_bounds__(NW* kWave, 2) k_attn_tile(KvAttnArgs a, const KvUnit* units, const int32_t* n_units,
                                                            int max_units, float* acc_out, float* ml_out) {
  constexpr int KS = D / 16, ND = D / 32, NJ = D / 64, kRows = 32 * NW;
  constexpr int kKBytes = 2 * KS * 1024, kVBytes = 4 * ND * 1024;  // fragments of a tile: 1 KB each
  constexpr int kBuf = kKBytes + kVBytes + 64;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // [2][K fragments, V fragments, TileMeta]
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  // the 16 keys of a tile that this wave decodes: K, V or (4 waves) both
  const int part = wave & 3;
  const bool does_k = NW == 4 || wave < 4, does_v = NW == 4 || wave >= 4;
  const int items = min(*n_units, max_units) * a.c.heads;
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int h = item % a.c.heads;
    const KvUnit u = units[item / a.c.heads];
    const int q0 = a.q_start[u.req], q_len = a.q_start[u.req + 1] - q0, kv_len = a.kv_len[u.req];
    const int rows = min(q_len * a.group - u.row, kRows);
    const int r = wave * 32 + col, row = u.row + r, tok = row / a.group;
    const bool in = r < rows && q0 + tok < a.total;
    const int limit = in ? kv_len - q_len + tok + 1 : 0x7FFFFFFF;  // keys that the row sees

    half8_t q[KS];
    float rowf = a.scale_log2;
    {
      const uint16_t* src = a.q + (long long)(q0 + tok) * a.q_row + (long long)(h * a.group + row % a.group) * a.q_head;
      uint4 raw[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s)
        raw[s] = in ? *reinterpret_cast<const uint4*>(src + 16 * ((s & ~1) + half) + 8 * (s & 1)) : uint4{0, 0, 0, 0};
      if constexpr (kBf16) {
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = max(top, max(word(raw[s], i) & 0x7FFFu, (word(raw[s], i) >> 16) & 0x7FFFu));
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
    // keys below `plain` need no mask in this wave, keys from `most` on do not matter to it
    const int first_row = u.row + min(wave * 32, rows), end_row = u.row + min((wave + 1) * 32, rows);
    const int plain = kv_len - q_len + first_row / a.group + 1;
    const int most = end_row > first_row ? kv_len - q_len + (end_row - 1) / a.group + 1 : 0;
    const int last = max(0, (u.kv_end - 1) >> a.c.b_shift);

    float m = kLowest, l = 0.0f, x = 0.0f;
    float16_t acc[ND];
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[n][e] = 0.0f;

    unsigned long long bad_seen = 0;
    Pages pages = load_pages(a, u.req, h, u.kv_begin >> a.c.b_shift, last, lane);
    if (u.kv_begin < u.kv_end) bad_seen = pages.bad;

    uint4 kr[NJ], vr[2];
    const auto load = [&](int pos, const Pages& p) {
      const int at = pos + 16 * part;
      const int id = __builtin_amdgcn_readlane(p.id, min(at >> a.c.b_shift, last) - p.first);
      const uint8_t* kb = a.c.data + ((long long)id * a.c.heads + h) * 2 * (a.c.B * D) + ((at & (a.c.B - 1)) >> 4) * (16 * D);
      const uint8_t* vb = kb + a.c.B * D;
      if (does_k) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) kr[j] = *reinterpret_cast<const uint4*>(kb + j * 1024 + lane * 16);
      }
      if (does_v) {
        // (head size 64: the upper lanes repeat the lower ones)
        const uint8_t* p0 = D == 128 ? vb + ((lane >> 4) & 1) * 1024 + half * 256 + (lane & 15) * 16
                                     : vb + ((lane >> 4) & 1) * 256 + (lane & 15) * 16;
        vr[0] = *reinterpret_cast<const uint4*>(p0);
        vr[1] = *reinterpret_cast<const uint4*>(p0 + 512);
      }
    };
    const auto store = [&](int pos, const Pages& p, char* buf) {
      const int at = pos + 16 * part, pg = min(at >> a.c.b_shift, last) - p.first;
      const bool bad = (p.bad >> pg) & 1;
      if (does_k) {
        // chunk c = 4 j + lane / 16 of token lane % 16
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int c = 4 * j + (lane >> 4);
          char* dst = buf + ((((part >> 1) * KS + (c & ~1)) * 64) + (c & 1) * 32 + (part & 1) * 16 + (lane & 15)) * 16;
          const uint2 w0 = kv_half4<kFmt>(kr[j].x), w1 = kv_half4<kFmt>(kr[j].y), w2 = kv_half4<kFmt>(kr[j].z),
                      w3 = kv_half4<kFmt>(kr[j].w);
          *reinterpret_cast<uint4*>(dst) = uint4{w0.x, w0.y, w1.x, w1.y};
          *reinterpret_cast<uint4*>(dst + 1024) = uint4{w2.x, w2.y, w3.x, w3.y};
        }
        if (lane == pg) {
          TileMeta* t = reinterpret_cast<TileMeta*>(buf + kKBytes + kVBytes);
          reinterpret_cast<float*>(&t->ks)[part] = p.ks;
          reinterpret_cast<float*>(&t->lv)[part] = p.lv;
          reinterpret_cast<float*>(&t->iv)[part] = p.iv;
          t->bad[part] = bad;
        }
      }
      if (does_v) {
        uint32_t keep[2] = {~0u, ~0u};
        if (kFmt == NSMLP_KV_E4M3 && (at + 16 > kv_len || bad)) {
          // codes past the end may be NaNs: a zero weight does not hide them
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int left = bad ? 0 : kv_len - (at + 8 * i + 4 * (D == 128 ? half : (lane >> 4) & 1));
            keep[i] = left >= 4 ? ~0u : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
          }
        }
        char* vbuf = buf + kKBytes + part * ND * 1024;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint2 lo = kv_half4<kFmt>(word(vr[0], i) & keep[0]), hi = kv_half4<kFmt>(word(vr[1], i) & keep[1]);
          const uint4 f = uint4{lo.x, lo.y, hi.x, hi.y};
          if constexpr (D == 128) {
            *reinterpret_cast<uint4*>(vbuf + (i * 64 + lane) * 16) = f;
          } else {
            if (lane < 32)
              *reinterpret_cast<uint4*>(vbuf + ((i >> 1) * 64 + ((lane >> 4) & 1) * 32 + (lane & 15) + 16 * (i & 1)) * 16) = f;
          }
        }
      }
    };

    // One tile's products.  kMasked: some rows do not see all of its keys.
    const auto tile = [&](auto masked, int pos, const char* buf) {
      constexpr bool kMasked = decltype(masked)::value;
      const half8_t* kf = reinterpret_cast<const half8_t*>(buf) + lane;
      const half8_t* vf = reinterpret_cast<const half8_t*>(buf + kKBytes) + lane;
      const TileMeta* t = reinterpret_cast<const TileMeta*>(buf + kKBytes + kVBytes);
      const float4_t ks = t->ks, lv = t->lv, iv = t->iv;
      float16_t s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[i][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) s[i] = mfma32(kf[(i * KS + k) * 64], q[k], s[i]);
      }
      // bit 8 i + e: whether the row sees key e of the lane's 8 among the tile's i-th 16
      uint32_t see = ~0u;
      if constexpr (kMasked) {
        see = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int n = min(max(limit - pos - 8 * i - 4 * half, 0), 4);
          see |= ((1u << n) - 1u) << (4 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) see = t->bad[i] != 0 ? see & ~(0xFFu << (8 * i)) : see;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[i][e] = (see >> (16 * i + e)) & 1 ? s[i][e] : -INFINITY;
      }
      uint4 w[4];
      float dl, dx;
      const auto weights = [&]() {
        dl = dx = 0.0f;
        float most_sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float g = ks[i] * rowf, c = lv[i] - m;
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) p[e] = exp2_fast(__builtin_fmaf(s[i >> 1][8 * (i & 1) + e], g, c));
          float share = iv[i];
          if constexpr (kMasked) {
            // a hidden key's weight is zero whatever its block's scales are
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = (see >> (8 * i + e)) & 1 ? p[e] : 0.0f;
            share = (see >> (8 * i)) & 0xFF ? share : 0.0f;
          }
          w[i] = uint4{pack_f16(p[0], p[1]), pack_f16(p[2], p[3]), pack_f16(p[4], p[5]), pack_f16(p[6], p[7])};
          const half2_t one = {(_Float16)1.0f, (_Float16)1.0f};
          float sum = __builtin_amdgcn_fdot2(as_half2(w[i].x), one, 0.0f, false);
          sum = __builtin_amdgcn_fdot2(as_half2(w[i].y), one, sum, false);
          sum = __builtin_amdgcn_fdot2(as_half2(w[i].z), one, sum, false);
          sum = __builtin_amdgcn_fdot2(as_half2(w[i].w), one, sum, false);
          most_sum = i == 0 ? sum : fmaxf(most_sum, sum);
          dl = __builtin_fmaf(sum, share, dl);
          if constexpr (kLse) dx = __builtin_fmaf(((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])), share, dx);
        }
        return most_sum;
      };
      sched_fence();  // the products' operands are not fetched further ahead than registers last
      const float sum = weights();
      if (__builtin_expect_with_probability(__any(sum > kSumLimit), 0, 0.999)) {
        float top = kLowest;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fmaf(max16(s[i >> 1], 8 * (i & 1)), ks[i] * rowf, lv[i]));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        top = ceilf(fmaxf(top, m));
        const float scale = exp2_fast(m - top);
        m = top;
        l *= scale, x *= scale;
#pragma unroll
        for (int n = 0; n < ND; ++n) acc[n] *= scale;
        (void)weights();
      }
      l += dl;
      if constexpr (kLse) x += dx;
      sched_fence();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < ND; ++n) acc[n] = mfma32(vf[(i * ND + n) * 64], as_h8(w[i]), acc[n]);
      sched_fence();
    };

    char* cur = lds;
    char* nxt = lds + kBuf;
    if (u.kv_begin < u.kv_end) {
      load(u.kv_begin, pages);
      store(u.kv_begin, pages, cur);
    }
    __syncthreads();
    int pos = u.kv_begin;
    const auto ahead = [&]() {  // the next tile's codes, before this one's products
      if (pos + kTileKeys < u.kv_end) {
        const int hi = min((pos + 2 * kTileKeys - 1) >> a.c.b_shift, last);
        if (hi - pages.first >= kWave) {
          pages = load_pages(a, u.req, h, (pos + kTileKeys) >> a.c.b_shift, last, lane);
          bad_seen |= pages.bad;
        }
        load(pos + kTileKeys, pages);
      }
    };
    const auto next = [&]() {
      if (pos + kTileKeys < u.kv_end) store(pos + kTileKeys, pages, nxt);
      __syncthreads();
      char* t = cur;
      cur = nxt, nxt = t;
      pos += kTileKeys;
    };
    // three loops, so that the accumulators stay where they are in each:
    // tiles that all rows see, tiles with hidden keys (or, from the first block
    // that is none, all that follow), tiles that only other waves need
    while (pos < u.kv_end && pos + kTileKeys <= plain && bad_seen == 0) {
      ahead();
      tile(std::false_type{}, pos, cur);
      next();
    }
    while (pos < u.kv_end && pos < most) {
      ahead();
      tile(std::true_type{}, pos, cur);
      next();
    }
    while (pos < u.kv_end) {
      ahead();
      next();
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
          for (int i = 0; i < 4; ++i) *reinterpret_cast<float4_t*>(acc_out + at * D + dim_of(g) + 4 * i) = piece(g, i, 1.0f);
        if (half == 0) *reinterpret_cast<float4_t*>(ml_out + 4 * at) = float4_t{m, l, x, 0.0f};
      } else {
        const long long at = (long long)(q0 + tok) * a.c.heads * a.group + h * a.group + row % a.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int g = 0; g < D / 32; ++g) {
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4_t p = piece(g, i, inv);
            o[2 * i] = to_out<kBf16>(p[0]) | (uint32_t)to_out<kBf16>(p[1]) << 16;
            o[2 * i + 1] = to_out<kBf16>(p[2]) | (uint32_t)to_out<kBf16>(p[3]) << 16;
          }
          uint4* dst = reinterpret_cast<uint4*>(a.out + at * D + dim_of(g));
          dst[0] = uint4{o[0], o[1], o[2], o[3]};
          dst[1] = uint4{o[4], o[5], o[6], o[7]};
        }
        if (kLse && half == 0) a.lse[at] = x == 0.0f ? -INFINITY : (m + log2f(x)) * 0.6931471805599453f;
      }
    }
  }
}

// ------------------------------------------------------------------ join --
// One wave per row whose keys were shared out: weights 2^(m_p - max m), in the
// order of the parts, so that the result does not depend on the schedule of
// the device.
template <int D, bool kBf16>
__global__ void __launch_bounds__(256) k_attn_join(KvAttnArgs a, const KvSplit* splits, const int32_t* n_splits,
                                                   int rows_of_unit, const float* acc_in, const float* ml_in) {
  constexpr int E = D / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int items = *n_splits * a.c.heads * rows_of_unit;
  for (int item = (int)blockIdx.x * 4 + (threadIdx.x >> 6); item < items; item += (int)gridDim.x * 4) {
    const int r = item % rows_of_unit, h = item / rows_of_unit % a.c.heads;
    const KvSplit sp = splits[item / rows_of_unit / a.c.heads];
    const int q0 = a.q_start[sp.req], q_len = a.q_start[sp.req + 1] - q0;
    const int full = sp.row + r, tok = q0 + full / a.group;
    if (full >= q_len * a.group || tok >= a.total) continue;
    const long long first = ((long long)sp.first * a.c.heads + h) * rows_of_unit + r;
    const long long step = (long long)a.c.heads * rows_of_unit;
    float top = kLowest;
    for (int p = lane; p < sp.parts; p += kWave) top = fmaxf(top, ml_in[4 * (first + p * step)]);
    top = wave_max(top);
    float l = 0.0f, x = 0.0f, o[E] = {};
#pragma unroll 4
    for (int p = 0; p < sp.parts; ++p) {
      const long long at = first + p * step;
      const float4_t ml = *reinterpret_cast<const float4_t*>(ml_in + 4 * at);
      const float w = exp2_fast(ml[0] - top);
      l += ml[1] * w, x += ml[2] * w;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += acc_in[at * D + lane * E + e] * w;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const long long at = (long long)tok * a.c.heads * a.group + h * a.group + full % a.group;
    if constexpr (E == 2)
      *reinterpret_cast<uint32_t*>(a.out + at * D + lane * 2) =
          to_out<kBf16>(o[0] * inv) | (uint32_t)to_out<kBf16>(o[1] * inv) << 16;
    else
      a.out[at * D + lane] = to_out<kBf16>(o[0] * inv);
    if (a.lse != nullptr && lane == 0) a.lse[at] = x == 0.0f ? -INFINITY : (top + log2f(x)) * 0.6931471805599453f;
  }
}

template <int D, int kFmt, bool kBf16, int NW, bool kLse>
void launch_tile(const KvAttnArgs& a, const KvUnit* units, hipStream_t s) {
  constexpr int kLds = 2 * ((D / 16 * 2 + D / 32 * 4) * 1024 + 64);
  static std::once_flag once;
  std::call_once(once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_attn_tile<D, kFmt, kBf16, NW, kLse>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
  });
  const unsigned grid = (unsigned)min((long long)a.s.max_units_b * a.c.heads, 65536LL);
  k_attn_tile<D, kFmt, kBf16, NW, kLse><<<dim3(grid), dim3(NW * kWave), kLds, s>>>(a, units, a.sched + 2, a.s.max_units_b,
                                                                                 a.acc_b, a.ml_b);
}

template <int D, int kFmt, bool kBf16>
void attention_typed(const KvAttnArgs& a, hipStream_t s) {
  const KvUnit* ua = reinterpret_cast<const KvUnit*>(a.sched + a.s.off_units_a);
  const KvUnit* ub = reinterpret_cast<const KvUnit*>(a.sched + a.s.off_units_b);
  const KvSplit* sa = reinterpret_cast<const KvSplit*>(a.sched + a.s.off_splits_a);
  const KvSplit* sb = reinterpret_cast<const KvSplit*>(a.sched + a.s.off_splits_b);
  auto grid = [&](long long units) { return dim3((unsigned)min(units * a.c.heads, 1024LL)); };
  auto join_grid = [&](long long splits, int rows) { return dim3((unsigned)min((splits * a.c.heads * rows + 3) / 4, 1024LL)); };
  k_attn_stream<D, kFmt, kBf16, 1><<<grid(a.s.max_units_a), dim3(kStreamThreads), 0, s>>>(a, ua, a.sched, a.s.max_units_a, a.s.rows_a,
                                                                                         a.acc_a, a.ml_a);
  if (a.s.max_splits_a > 0)
    k_attn_join<D, kBf16><<<join_grid(a.s.max_splits_a, a.s.rows_a), dim3(256), 0, s>>>(a, sa, a.sched + 1, a.s.rows_a,
                                                                                       a.acc_a, a.ml_a);
  if (a.list_b) {
    if (a.s.rows_b == 256) a.lse != nullptr ? launch_tile<D, kFmt, kBf16, 8, true>(a, ub, s) : launch_tile<D, kFmt, kBf16, 8, false>(a, ub, s);
    else a.lse != nullptr ? launch_tile<D, kFmt, kBf16, 4, true>(a, ub, s) : launch_tile<D, kFmt, kBf16, 4, false>(a, ub, s);
    if (a.s.max_splits_b > 0)
      k_attn_join<D, kBf16><<<join_grid(a.s.max_splits_b, a.s.rows_b), dim3(256), 0, s>>>(a, sb, a.sched + 3, a.s.rows_b,
                                                                                         a.acc_b, a.ml_b);
  }
}

}  // namespace

size_t kv_attn_partial_floats(const KvSchedule& s, int kv_heads, int D, size_t (&off)[4]) {
  size_t at = 0;
  const size_t ra = (size_t)s.max_parts_a * kv_heads * s.rows_a, rb = (size_t)s.max_parts_b * kv_heads * s.rows_b;
  off[0] = at, at += ra * D;
  off[1] = at, at += ra * 4;
  off[2] = at, at += rb * D;
  off[3] = at, at += rb * 4;
  return at;
}

void launch_kv_attention(const KvAttnArgs& a, bool bf16, hipStream_t s) {
  NSMLP_KV_BY_TYPE(attention_typed, a, bf16, s);
}

}  // namespace nsmlp
