// Bookkeeping of the paged 8-bit K/V cache: a step's plan (block tables, slot
// maps, the attention's work lists), commit, append and read.
#include "nsmlp_kv.h"

#include <mutex>

namespace nsmlp {

namespace {

// ------------------------------------------------------------------ plan --
// Every workgroup scans all requests (a few KB, from L2) into LDS, so that no
// workgroup waits for another; then each writes its share of the slots and of
// the work lists.  Requests are taken in order: request r needs
//   need = ceil((cached + fresh) / B) - ceil(cached / B)
// blocks, the ring's entries head + (sum of need before r) ...; it is refused
// (no slots, kv_len 0, lengths unchanged) where its blocks exceed the table's
// width or the running sum the free count.
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(v, d, kWave);
    if (lane >= d) v += o;
  }
  return v;
}

// Exclusive sums of N values over the workgroup's threads, totals in `total`.
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*wsum)[kPlanWaves], int tid) {
  const int lane = tid & (kWave - 1), wave = tid >> 6;
  int inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    inc[i] = wave_scan(v[i], lane);
    if (lane == kWave - 1) wsum[i][wave] = inc[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int before = 0, all = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int x = wsum[i][w];
      before += w < wave ? x : 0;
      all += x;
    }
    v[i] = before + inc[i] - v[i];
    total[i] = all;
  }
  __syncthreads();
}

__device__ __forceinline__ int clip_len(int v) { return min(max(v, 0), 1 << 29); }

constexpr int kPer = kKvMaxRequests / kPlanThreads;

// keys per part, so that about `target` units share the list's `work` keys
__device__ __forceinline__ int part_keys(long long work, int target, int least) {
  if (target <= 0) return 1 << 30;  // more than any request's
  const long long each = (work + target - 1) / target;
  const long long up = (each + 127) / 128 * 128;
  return up < least ? least : up > (1 << 30) ? 1 << 30 : (int)up;
}

__global__ void __launch_bounds__(kPlanThreads) k_kv_plan(KvPlanArgs a) {
  extern __shared__ __attribute__((aligned(16))) int lds[];
  __shared__ int wsum[4][kPlanWaves];
  __shared__ long long wsum2[2][kPlanWaves];
  __shared__ int refused_s;
  int* q_start = lds;           // [R + 1]
  int* base = q_start + a.R + 1;  // [R] blocks granted before the request; -1: refused
  int* first = base + a.R;        // [R] first unit of its list
  int* split = first + a.R;       // [R] first split tile of its list
  int* partial = split + a.R;     // [R] first partial
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int per = (a.R + kPlanThreads - 1) / kPlanThreads;
  const int r0 = tid * per;
  const unsigned N = (unsigned)a.num_blocks;
  const int head = (int)((unsigned)a.state[0] % N), count = min(max(a.state[1], 0), a.num_blocks);
  if (tid == 0) refused_s = 0;

  int cached[kPer], fresh[kPer], need[kPer];
  int sum[2] = {0, 0}, total[2];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i;
    const bool in = i < per && r < a.R;
    cached[i] = in ? clip_len(a.cached[r]) : 0;
    fresh[i] = in ? min(max(a.fresh[r], 0), 1 << 28) : 0;
    const int have = (cached[i] + a.B - 1) >> a.b_shift, tot = (cached[i] + fresh[i] + a.B - 1) >> a.b_shift;
    need[i] = tot <= a.max_blocks ? tot - have : -1;  // -1: longer than the table
    sum[0] += fresh[i];
    sum[1] += max(need[i], 0);
  }
  block_scan(sum, total, wsum, tid);
  // granted requests, and the work of either list
  int at = sum[0], used = sum[1], refused = 0, kv[kPer];
  long long work[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i;
    if (i < per && r < a.R) {
      const int n = max(need[i], 0);
      const bool ok = need[i] >= 0 && (n == 0 || used + n <= count) && fresh[i] <= a.max_new;
      q_start[r] = at;
      base[r] = ok ? used : -1;
      kv[i] = ok ? cached[i] + fresh[i] : 0;
      refused += !ok && fresh[i] > 0;
      used += n;
      at += fresh[i];
      const long long rows = (long long)fresh[i] * a.group;
      if (rows > a.s.rows_a) work[1] += (rows + a.s.rows_b - 1) / a.s.rows_b * kv[i];
      else if (rows > 0) work[0] += kv[i];
    } else {
      kv[i] = 0;
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const long long w = wave_sum(work[i]);
    if (lane == 0) wsum2[i][wave] = w;
  }
  if (refused) atomicAdd(&refused_s, refused);
  if (tid == 0) q_start[a.R] = total[0];
  __syncthreads();
  long long all[2] = {0, 0};
  for (int w = 0; w < kPlanWaves; ++w) {
    all[0] += wsum2[0][w];
    all[1] += wsum2[1][w];
  }
  const int keys_a = part_keys(all[0], a.s.target_a, a.s.min_a), keys_b = part_keys(all[1], a.s.target_b, a.s.min_b);
  // units of each request: tiles of rows times parts of its keys
  int cnt[4] = {0, 0, 0, 0}, cnt_total[4];  // units a, units b, split tiles a, split tiles b
  int parts_b_sum[1] = {0}, parts_b_total[1];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const long long rows = (long long)fresh[i] * a.group;
    if (rows == 0) continue;
    if (rows > a.s.rows_a) {
      const int tiles = (int)((rows + a.s.rows_b - 1) / a.s.rows_b), parts = max(1, (kv[i] + keys_b - 1) / keys_b);
      cnt[1] += tiles * parts;
      if (parts > 1) {
        cnt[3] += tiles;
        parts_b_sum[0] += tiles * parts;
      }
    } else {
      const int parts = max(1, (kv[i] + keys_a - 1) / keys_a);
      cnt[0] += parts;
      if (parts > 1) cnt[2] += 1;
    }
  }
  int parts_a_sum[1] = {0}, parts_a_total[1];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const long long rows = (long long)fresh[i] * a.group;
    if (rows > 0 && rows <= a.s.rows_a) {
      const int parts = max(1, (kv[i] + keys_a - 1) / keys_a);
      if (parts > 1) parts_a_sum[0] += parts;
    }
  }
  block_scan(cnt, cnt_total, wsum, tid);
  block_scan(parts_a_sum, parts_a_total, wsum, tid);
  block_scan(parts_b_sum, parts_b_total, wsum, tid);
  int ua = cnt[0], ub = cnt[1], sa = cnt[2], sb = cnt[3], pa = parts_a_sum[0], pb = parts_b_sum[0];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i;
    if (i >= per || r >= a.R) continue;
    const long long rows = (long long)fresh[i] * a.group;
    if (rows > a.s.rows_a) {
      const int tiles = (int)((rows + a.s.rows_b - 1) / a.s.rows_b), parts = max(1, (kv[i] + keys_b - 1) / keys_b);
      first[r] = ub, split[r] = sb, partial[r] = pb;
      ub += tiles * parts;
      if (parts > 1) sb += tiles, pb += tiles * parts;
    } else {
      const int parts = rows == 0 ? 0 : max(1, (kv[i] + keys_a - 1) / keys_a);
      first[r] = ua, split[r] = sa, partial[r] = pa;
      ua += parts;
      if (parts > 1) sa += 1, pa += parts;
    }
    if (blockIdx.x == 0) {
      a.q_start[r] = q_start[r];
      a.kv_len[r] = kv[i];
      a.next[r] = base[r] >= 0 ? cached[i] + fresh[i] : cached[i];
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.q_start[a.R] = total[0];
    // blocks used: the needs of granted requests (a refused one takes none)
    a.info[2] = refused_s;
    a.info[3] = total[0];
    a.sched[0] = min(cnt_total[0], a.s.max_units_a);
    a.sched[1] = min(cnt_total[2], a.s.max_splits_a);
    a.sched[2] = min(cnt_total[1], a.s.max_units_b);
    a.sched[3] = min(cnt_total[3], a.s.max_splits_b);
  }
  {
    int granted[1] = {0}, granted_total[1];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < per && r0 + i < a.R && base[r0 + i] >= 0) granted[0] += max(need[i], 0);
    block_scan(granted, granted_total, wsum, tid);  // its barriers also publish the LDS arrays
    if (blockIdx.x == 0 && tid == 0) {
      a.info[0] = (int)(((unsigned)head + (unsigned)granted_total[0]) % N);
      a.info[1] = count - granted_total[0];
    }
  }
  // slots: one thread per token; a block's first token also writes its entry
  for (long long t = (long long)blockIdx.x * kPlanThreads + tid; t < a.total; t += (long long)gridDim.x * kPlanThreads) {
    int lo = 0, hi = a.R;  // the last request with q_start <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (q_start[mid] <= t) lo = mid;
      else hi = mid;
    }
    long long slot = -1;
    if (t < q_start[a.R] && base[lo] >= 0) {
      const int c = clip_len(a.cached[lo]);
      const int have = (c + a.B - 1) >> a.b_shift, p = c + (int)t - q_start[lo], j = p >> a.b_shift;
      int32_t* entry = a.table + (long long)lo * a.max_blocks + j;
      int id;
      if (j < have) {
        id = *entry;
      } else {
        id = a.ring[((unsigned)head + (unsigned)(base[lo] + j - have)) % N];
        if ((p & (a.B - 1)) == 0) *entry = id;
      }
      if (id >= 0 && id < a.num_blocks) slot = ((long long)id << a.b_shift) + (p & (a.B - 1));
    }
    a.slots[t] = slot;
  }
  // work lists: one wave per request
  KvUnit* units_a = reinterpret_cast<KvUnit*>(a.sched + a.s.off_units_a);
  KvUnit* units_b = reinterpret_cast<KvUnit*>(a.sched + a.s.off_units_b);
  KvSplit* splits_a = reinterpret_cast<KvSplit*>(a.sched + a.s.off_splits_a);
  KvSplit* splits_b = reinterpret_cast<KvSplit*>(a.sched + a.s.off_splits_b);
  for (int r = (int)blockIdx.x * kPlanWaves + wave; r < a.R; r += (int)gridDim.x * kPlanWaves) {
    const int q = q_start[r + 1] - q_start[r];
    if (q == 0) continue;
    const int c = clip_len(a.cached[r]), len = base[r] >= 0 ? c + q : 0;
    const long long rows = (long long)q * a.group;
    const bool b = rows > a.s.rows_a;
    const int per_tile = b ? a.s.rows_b : a.s.rows_a, keys = b ? keys_b : keys_a;
    const int tiles = (int)((rows + per_tile - 1) / per_tile), parts = max(1, (len + keys - 1) / keys);
    KvUnit* units = b ? units_b : units_a;
    KvSplit* splits = b ? splits_b : splits_a;
    const int max_units = b ? a.s.max_units_b : a.s.max_units_a, max_splits = b ? a.s.max_splits_b : a.s.max_splits_a,
              max_parts = b ? a.s.max_parts_b : a.s.max_parts_a;
    for (int i = lane; i < tiles * parts; i += kWave) {
      // the last tile sees the most keys: it goes first
      const int tile = tiles - 1 - i / parts, part = i % parts;
      const int last = (int)min((long long)q, ((long long)(tile + 1) * per_tile + a.group - 1) / a.group);
      const int keys_seen = max(0, len - q + last);  // of the tile's last row
      const int each = ((keys_seen + parts - 1) / parts + 63) & ~63;
      KvUnit u;
      u.req = r;
      u.row = tile * per_tile;
      u.kv_begin = min(part * each, keys_seen);
      u.kv_end = min((part + 1) * each, keys_seen);
      u.part = parts > 1 ? partial[r] + i : -1;
      u.pad[0] = u.pad[1] = u.pad[2] = 0;
      if (first[r] + i < max_units && u.part < max_parts) units[first[r] + i] = u;
      if (parts > 1 && part == 0 && split[r] + i / parts < max_splits)
        splits[split[r] + i / parts] = KvSplit{r, u.row, u.part, parts};
    }
  }
}

// Lengths, ring state and (for finished requests) the table after a step.  A
// finished request's blocks return to the ring's end in the order of requests
// and of their tables; one workgroup, as the order is a running sum.
__global__ void __launch_bounds__(kPlanThreads) k_kv_commit(KvCommitArgs a) {
  __shared__ int wsum[1][kPlanWaves];
  const int tid = threadIdx.x;
  const int per = (a.R + kPlanThreads - 1) / kPlanThreads, r0 = tid * per;
  const unsigned N = (unsigned)a.num_blocks;
  const int* from = a.info != nullptr ? a.info : a.state;
  const int head = (int)((unsigned)from[0] % N), count = min(max(from[1], 0), a.num_blocks);
  int mine[1] = {0}, total[1];
  for (int i = 0; i < per; ++i) {
    const int r = r0 + i;
    if (r >= a.R) break;
    const int len = a.next != nullptr ? a.next[r] : a.cached[r];
    if (a.finished != nullptr && a.finished[r] != 0)
      mine[0] += min((max(len, 0) + a.B - 1) >> a.b_shift, a.max_blocks);
  }
  block_scan(mine, total, wsum, tid);
  int at = mine[0];
  for (int i = 0; i < per; ++i) {
    const int r = r0 + i;
    if (r >= a.R) break;
    const int len = a.next != nullptr ? a.next[r] : a.cached[r];
    if (a.finished != nullptr && a.finished[r] != 0) {
      const int n = min((max(len, 0) + a.B - 1) >> a.b_shift, a.max_blocks);
      for (int j = 0; j < n; ++j) {
        // never more than the ring holds: a table with an id twice cannot push the ring past its size
        if (count + at + j < a.num_blocks)
          a.ring[((unsigned)head + (unsigned)(count + at + j)) % N] = a.table[(long long)r * a.max_blocks + j];
        a.table[(long long)r * a.max_blocks + j] = -1;
      }
      at += n;
      a.cached[r] = 0;
    } else {
      a.cached[r] = len;
    }
  }
  if (tid == 0) {
    a.state[0] = head;
    a.state[1] = min(count + total[0], a.num_blocks);
  }
}

// ---------------------------------------------------------------- append --
// One wave per (run, head, K or V): a run is the tokens of one block, which
// stand next to each other in the call.  The wave of a run's first token does
// it; the others leave.  Two passes over the run's rows (the second from the
// caches): the largest magnitude, then the codes.
constexpr int kAppendThreads = 256;

template <bool kBf16>
__device__ __forceinline__ float in_value(uint16_t h) {
  if constexpr (kBf16) return __uint_as_float((uint32_t)h << 16);
  else return h2f(h);
}

template <int D, int kFmt, bool kBf16>
__global__ void __launch_bounds__(kAppendThreads) k_kv_append(KvAppendArgs a) {
  constexpr int kChunks = D / 16, kTok = kWave / kChunks;  // 16-dim pieces of a token, tokens of a pass
  const int lane = threadIdx.x & (kWave - 1);
  const long long item = (long long)blockIdx.x * (kAppendThreads / kWave) + (threadIdx.x >> 6);
  const int two_heads = 2 * a.c.heads;
  const int t = (int)(item / two_heads), hk = (int)(item % two_heads), h = hk >> 1;
  const bool is_v = hk & 1;
  if (t >= a.n) return;
  const long long limit = (long long)a.c.num_blocks * a.c.B;
  const long long slot = a.slots[t];
  if (slot < 0 || slot >= limit) return;
  const long long blk = slot >> a.c.b_shift;
  if (t > 0) {
    const long long prev = a.slots[t - 1];
    if (prev >= 0 && prev < limit && prev == slot - 1 && (prev >> a.c.b_shift) == blk) return;
  }
  const int o0 = (int)(slot & (a.c.B - 1));  // first new offset
  // run length: B <= 64 lanes look at the following tokens
  const long long mine = t + lane < a.n && lane < a.c.B - o0 ? a.slots[t + lane] : -1;
  const unsigned long long same = __ballot(mine == slot + lane);
  const int n = same == ~0ull ? 64 : __builtin_ctzll(~same);

  const uint16_t* x = is_v ? a.v + (long long)t * a.v_row + (long long)h * a.v_head
                           : a.k + (long long)t * a.k_row + (long long)h * a.k_head;
  const long long row = is_v ? a.v_row : a.k_row;
  float* sp = a.c.scale + (blk * a.c.heads + h) * 2 + (is_v ? 1 : 0);
  const float s_old = o0 == 0 ? 0.0f : *sp;
  uint8_t* dst = a.c.data + ((blk * a.c.heads + h) * 2 + (is_v ? 1 : 0)) * (long long)(a.c.B * D);

  // largest magnitude, as bits (a NaN or infinity is above every finite value)
  const int tl = lane / kChunks, c = lane % kChunks;
  uint32_t top = 0;
  for (int i = tl; i < n; i += kTok) {
    const uint4* p = reinterpret_cast<const uint4*>(x + i * row + c * 16);
    const uint4 u0 = p[0], u1 = p[1];
    const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, max(w[j] & 0x7FFFu, (w[j] >> 16) & 0x7FFFu));
  }
#pragma unroll
  for (int m = kWave / 2; m >= 1; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, kWave));
  const float need = kv_scale_of<kFmt>(in_value<kBf16>((uint16_t)top));
  // a NaN on either side stays until the block is started anew
  const float s_new = need != need || s_old != s_old ? __uint_as_float(0x7FC00000u) : fmaxf(s_old, need);
  const bool recode = o0 > 0 && s_new != s_old;
  if (lane == 0) *sp = s_new;

  if (!is_v) {
    if (recode) {
      for (int i = tl; i < o0; i += kTok) {
        uint32_t* q = reinterpret_cast<uint32_t*>(dst + kv_k_off(D, i, c * 16));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w = q[j];
          uint32_t r = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            r |= kv_encode1<kFmt>(kv_decode1<kFmt>((w >> (8 * b)) & 0xFFu) * s_old / s_new) << (8 * b);
          q[j] = r;
        }
      }
    }
    for (int i = tl; i < n; i += kTok) {
      const uint4* p = reinterpret_cast<const uint4*>(x + i * row + c * 16);
      const uint4 u0 = p[0], u1 = p[1];
      const uint32_t w[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
      uint32_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        r[j] = kv_encode1<kFmt>(in_value<kBf16>((uint16_t)w[2 * j]) / s_new) |
               kv_encode1<kFmt>(in_value<kBf16>((uint16_t)(w[2 * j] >> 16)) / s_new) << 8 |
               kv_encode1<kFmt>(in_value<kBf16>((uint16_t)w[2 * j + 1]) / s_new) << 16 |
               kv_encode1<kFmt>(in_value<kBf16>((uint16_t)(w[2 * j + 1] >> 16)) / s_new) << 24;
      }
      *reinterpret_cast<uint4*>(dst + kv_k_off(D, o0 + i, c * 16)) = uint4{r[0], r[1], r[2], r[3]};
    }
  } else {
    // pieces of 4 tokens by 4 dims, 16 bytes; the wave owns the block's V, so
    // a piece's other tokens are read and written back
    constexpr int kPieces = D / 4, kGroups = kWave / kPieces;
    const int gl = lane / kPieces, d0 = lane % kPieces * 4;
    const int g_end = (o0 + n + 3) >> 2;
    for (int g = (recode ? 0 : o0 >> 2) + gl; g < g_end; g += kGroups) {
      uint4* q = reinterpret_cast<uint4*>(dst + kv_v_off(D, 4 * g, d0));
      const bool all_new = 4 * g >= o0 && 4 * g + 4 <= o0 + n;
      uint4 old = uint4{0, 0, 0, 0};
      if (!all_new) old = *q;
      uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const int off = 4 * g + tt;
        if (off >= o0 && off < o0 + n) {
          const uint2 u = *reinterpret_cast<const uint2*>(x + (off - o0) * row + d0);
          const uint32_t e[2] = {u.x, u.y};
#pragma unroll
          for (int d = 0; d < 4; ++d)
            w[d] = (w[d] & ~(0xFFu << (8 * tt))) |
                   kv_encode1<kFmt>(in_value<kBf16>((uint16_t)(e[d >> 1] >> (16 * (d & 1)))) / s_new) << (8 * tt);
        } else if (off < o0 && recode) {
#pragma unroll
          for (int d = 0; d < 4; ++d)
            w[d] = (w[d] & ~(0xFFu << (8 * tt))) |
                   kv_encode1<kFmt>(kv_decode1<kFmt>((w[d] >> (8 * tt)) & 0xFFu) * s_old / s_new) << (8 * tt);
        }
      }
      *q = uint4{w[0], w[1], w[2], w[3]};
    }
  }
}

// ------------------------------------------------------------------ read --
// One thread per 8 dims of a (slot, head): values code * scale, rounded once.
template <int D, int kFmt, bool kBf16>
__global__ void __launch_bounds__(256) k_kv_read(KvReadArgs a) {
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int per = D / 8;
  const int d0 = (int)(item % per) * 8;
  const long long th = item / per;
  const int h = (int)(th % a.c.heads);
  const long long t = th / a.c.heads;
  if (t >= a.n) return;
  const long long slot = a.slots[t];
  uint32_t out[2][4] = {};
  if (slot >= 0 && slot < (long long)a.c.num_blocks * a.c.B) {
    const long long bh = (slot >> a.c.b_shift) * a.c.heads + h;
    const int off = (int)(slot & (a.c.B - 1));
    const uint8_t* kb = a.c.data + bh * 2 * (long long)(a.c.B * D);
    const uint8_t* vb = kb + a.c.B * D;
    const float ks = a.c.scale[bh * 2], vs = a.c.scale[bh * 2 + 1];
    const uint2 kw = *reinterpret_cast<const uint2*>(kb + kv_k_off(D, off, d0));
    const uint8_t* vp = vb + kv_v_off(D, off, d0);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const uint32_t kc = ((d < 4 ? kw.x : kw.y) >> (8 * (d & 3))) & 0xFFu;
      const float kx = kv_decode1<kFmt>(kc) * ks, vx = kv_decode1<kFmt>(vp[4 * d]) * vs;
      uint32_t kh, vh;
      if constexpr (kBf16) {
        kh = __builtin_bit_cast(uint16_t, (__bf16)kx), vh = __builtin_bit_cast(uint16_t, (__bf16)vx);
      } else {
        kh = f2h(kx), vh = f2h(vx);
      }
      out[0][d >> 1] |= kh << (16 * (d & 1));
      out[1][d >> 1] |= vh << (16 * (d & 1));
    }
  }
  const long long o = (t * a.c.heads + h) * D + d0;
  *reinterpret_cast<uint4*>(a.k + o) = uint4{out[0][0], out[0][1], out[0][2], out[0][3]};
  *reinterpret_cast<uint4*>(a.v + o) = uint4{out[1][0], out[1][1], out[1][2], out[1][3]};
}

template <template <int, int, bool> class L, class A>
void by_type(const A& a, bool bf16, hipStream_t s) {
  const bool i8 = a.c.fmt == NSMLP_KV_INT8, d128 = a.c.D == 128;
  if (d128) {
    if (i8) bf16 ? L<128, NSMLP_KV_INT8, true>::go(a, s) : L<128, NSMLP_KV_INT8, false>::go(a, s);
    else bf16 ? L<128, NSMLP_KV_E4M3, true>::go(a, s) : L<128, NSMLP_KV_E4M3, false>::go(a, s);
  } else {
    if (i8) bf16 ? L<64, NSMLP_KV_INT8, true>::go(a, s) : L<64, NSMLP_KV_INT8, false>::go(a, s);
    else bf16 ? L<64, NSMLP_KV_E4M3, true>::go(a, s) : L<64, NSMLP_KV_E4M3, false>::go(a, s);
  }
}

template <int D, int kFmt, bool kBf16>
struct AppendLaunch {
  static void go(const KvAppendArgs& a, hipStream_t s) {
    const long long waves = (long long)a.n * a.c.heads * 2, per = kAppendThreads / kWave;
    k_kv_append<D, kFmt, kBf16><<<dim3((unsigned)((waves + per - 1) / per)), dim3(kAppendThreads), 0, s>>>(a);
  }
};
template <int D, int kFmt, bool kBf16>
struct ReadLaunch {
  static void go(const KvReadArgs& a, hipStream_t s) {
    const long long items = (long long)a.n * a.c.heads * (D / 8);
    k_kv_read<D, kFmt, kBf16><<<dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s>>>(a);
  }
};

}  // namespace

void launch_kv_append(const KvAppendArgs& a, bool bf16, hipStream_t s) { by_type<AppendLaunch>(a, bf16, s); }
void launch_kv_read(const KvReadArgs& a, bool bf16, hipStream_t s) { by_type<ReadLaunch>(a, bf16, s); }

KvSchedule kv_schedule(int requests, int total, int max_new, int group, int kv_heads) {
  (void)max_new;
  KvSchedule s;
  s.rows_a = 16;
  s.rows_b = 16;
  const long long tiles_b = ((long long)total * group + s.rows_b - 1) / s.rows_b + requests;
  s.target_a = (1024 + kv_heads - 1) / kv_heads;
  s.target_b = tiles_b * kv_heads >= 2048 ? 0 : (1024 + kv_heads - 1) / kv_heads;
  s.min_a = 256;
  s.min_b = 512;
  // parts > 1 only where a request's keys exceed a part, so split units are at
  // most twice the work over the keys of a part, and split tiles at most it
  s.max_parts_a = 2 * s.target_a, s.max_parts_b = 2 * s.target_b;
  s.max_splits_a = s.target_a, s.max_splits_b = s.target_b;
  s.max_units_a = requests + s.max_parts_a;
  s.max_units_b = (int)tiles_b + s.max_parts_b;
  const long long unit = sizeof(KvUnit) / 4, split = sizeof(KvSplit) / 4;
  s.off_units_a = kKvHeaderInts;
  s.off_units_b = s.off_units_a + unit * s.max_units_a;
  s.off_splits_a = s.off_units_b + unit * s.max_units_b;
  s.off_splits_b = s.off_splits_a + split * s.max_splits_a;
  s.ints = s.off_splits_b + split * s.max_splits_b;
  return s;
}

void launch_kv_plan(const KvPlanArgs& a, hipStream_t s) {
  static std::once_flag once;
  constexpr int kMost = (5 * kKvMaxRequests + 1) * (int)sizeof(int);
  std::call_once(once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_kv_plan), hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
  });
  int groups = max((a.total + 2047) / 2048, (a.R + 63) / 64);
  groups = min(max(groups, 1), 64);
  k_kv_plan<<<dim3(groups), dim3(kPlanThreads), (5 * a.R + 1) * sizeof(int), s>>>(a);
}

void launch_kv_commit(const KvCommitArgs& a, hipStream_t s) {
  k_kv_commit<<<dim3(1), dim3(kPlanThreads), 0, s>>>(a);
}

}  // namespace nsmlp
