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
// width, its new tokens max_new, or the running sum the free count.  The ring
// moves on by the blocks granted, so what the first two refuse is in no sum;
// past the free count every later request that needs a block is refused too.
//
// What bounds it: latency (8 requests 6.5 us, 300 with 6513 tokens 10 us, 4096
// with 73470 tokens 14 us).  8 requests write 224 bytes, 4096 requests 0.7 MB; a
// step is a chain of one load of the lengths, two scans, one load of the
// ring's entries and the stores.  Sums within a wave go through DPP adds (a
// few cycles each; exchanges through LDS took most of the time before), the
// waves' sums meet in LDS once per scan, and the workgroup is no wider than
// the requests need: 64 threads need no barrier between waves at all.
__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0 -> 1, 2 -> 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // rows 0, 1 -> 2, 3
  return v;
}

// Exclusive sums of N values over the workgroup's threads, totals in `total`.
template <int N, int kThreads>
__device__ __forceinline__ void block_scan(int (&v)[N], int (&total)[N], int (*wsum)[16], int tid) {
  constexpr int kWaves = kThreads / kWave;
  const int lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) inc[i] = wave_scan(v[i]);
  if constexpr (kWaves == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) total[i] = __builtin_amdgcn_readlane(inc[i], kWave - 1), v[i] = inc[i] - v[i];
  } else {
    if (lane == kWave - 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) wsum[i][wave] = inc[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int all = wave_scan(lane < kWaves ? wsum[i][lane & 15] : 0);
      total[i] = __builtin_amdgcn_readlane(all, kWaves - 1);
      v[i] = inc[i] - v[i] + (wave == 0 ? 0 : __builtin_amdgcn_readlane(all, wave == 0 ? 0 : wave - 1));
    }
    __syncthreads();
  }
}

__device__ __forceinline__ int clip_len(int v) { return min(max(v, 0), 1 << 29); }

// list a counts keys in pieces of 64; a request without any takes one piece,
// so that its rows are somebody's
constexpr int kLeastShare = 4;     // pieces: 256 keys are worth a workgroup
// Keys per part of list b, L.  A part costs its rows' fp32 sums written and read
// back, about what kPartCost keys' products cost where the tile is full of rows.
// With w keys of work per CU in all, the CUs take w (1 + cost / L) and the longest
// part L; the two meet at `meet`.  Tiles with few rows are those of many short
// requests: their parts cost little, and as nobody sorts them by length, the
// last to end is what a smaller L shortens: w cost / L + L / 4 is least at `even`.
// List a's keys count half, as the parts run next to them on the same CUs (a
// prompt's 387 tokens next to 20 decodes: 39 us without, 32 with).
// Costs of 128 and 512 over 25 drawn prompts, drafts and mixed steps: 0.2% longer
// and 1% shorter calls on average, single ones 9% shorter to 8% longer and 20%
// shorter to 9% longer; least parts of 96 and 384: 0.7% and 0.8% longer on average.
constexpr float kPartCost = 256.0f, kLeastPart = 192.0f;

// 1 / L of a request with `rows` rows in `tiles` tiles.  (Parts are counted in
// one place and listed in another: no contraction, so that both get the same.)
__device__ __forceinline__ float parts_per_key(float w, int rows, int tiles, int rows_b) {
#pragma clang fp contract(off)
  const float fill = (float)rows / (float)(tiles * rows_b), cost = kPartCost * fill;
  const float meet = 0.5f * (w + sqrtf(w * (w + 4.0f * cost)));
  const float even = 2.0f * sqrtf(w * cost) / fmaxf(1.0f - fill, 1e-3f);
  return 1.0f / fmaxf(fmaxf(0.5f * w, kLeastPart), fminf(meet, even));
}

// keys that the last row of a tile of list b sees, of a request with q new tokens and len keys
__device__ __forceinline__ int tile_keys(int tile, int q, int len, int rows_b, int group) {
  const int last = min(q, (int)(((unsigned)(tile + 1) * (unsigned)rows_b + group - 1) / (unsigned)group));
  return max(0, len - q + last);
}
// and the sum of that over the request's tiles, or a little more
__device__ __forceinline__ long long work_of(int tiles, int q, int len, int rows_b, int group) {
  if (len <= 0) return 0;
  return (long long)tiles * (len - q) + (long long)(tiles - 1) * tiles / 2 * rows_b / group + tiles + q;
}
// parts of a tile: 1 below 1.35 L keys, at most 1.5 keys / L else
__device__ __forceinline__ int parts_of(int seen, float per_key) {
#pragma clang fp contract(off)
  return max(1, (int)((float)seen * per_key + 0.65f));
}

// Which list a request is in.  Without a list b its rows are list a's however
// many they are: then it is longer than max_new, refused, and its rows are only
// to be filled (or the step's total is less than the requests' sum).
__device__ __forceinline__ bool in_list_b(const KvPlanArgs& a, int rows) { return a.s.list_b && rows > kKvRowsA; }

__device__ __forceinline__ int pieces_of(int keys) { return max(1, (keys + 63) >> 6); }

constexpr int kPlanSums = 6;

template <int kThreads, int kPer>
__global__ void __launch_bounds__(kThreads) k_kv_plan(KvPlanArgs a) {
  extern __shared__ __attribute__((aligned(16))) int lds[];
  __shared__ int wsum[kPlanSums][16];
  int* q_start = lds;             // [R + 1]
  int* base = q_start + a.R + 1;  // [R] blocks granted before the request; -1: refused
  int* first = base + a.R;        // [R] first unit of its list
  int* split = first + a.R;       // [R] list b: first split tile; list a: pieces before the request
  int* partial = split + a.R;     // [R] first partial
  int* len_s = partial + a.R;     // [R] cached tokens
  kernarg_warm<sizeof(KvPlanArgs)>();
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int per = kPer == 1 ? 1 : (a.R + kThreads - 1) / kThreads;
  const int r0 = tid * per;
  const unsigned N = (unsigned)a.num_blocks;

  int cached[kPer], fresh[kPer], need[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i;
    const bool in = i < per && r < a.R;
    cached[i] = in ? clip_len(a.cached[r]) : 0;
    fresh[i] = in ? min(max(a.fresh[r], 0), 1 << 28) : 0;
  }
  const int head = (int)((unsigned)a.state[0] % N), count = min(max(a.state[1], 0), a.num_blocks);
  int sum[2] = {0, 0}, total[2];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int have = (cached[i] + a.B - 1) >> a.b_shift, tot = (cached[i] + fresh[i] + a.B - 1) >> a.b_shift;
    need[i] = tot <= a.max_blocks && fresh[i] <= a.max_new ? tot - have : -1;  // -1: longer than the table or max_new
    sum[0] += fresh[i];
    sum[1] += max(need[i], 0);
  }
  block_scan<2, kThreads>(sum, total, wsum, tid);
  // granted requests; list a's pieces, and list b's work (tiles of rows times
  // keys) in three summands of 20 bits (1024 of them stay in 30)
  int at = sum[0], used = sum[1], kv[kPer], tiles[kPer];  // tiles -1: list a
  long long work = 0;
  int cnt[kPlanSums] = {};  // units a, units b, splits b, partials a, partials b, blocks granted
  int sums[5] = {}, sums_total[5];  // pieces of list a, work of list b, refused
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i;
    const bool in = i < per && r < a.R;
    const int n = max(need[i], 0);
    const bool ok = need[i] >= 0 && (n == 0 || used + n <= count);
    kv[i] = in && ok ? cached[i] + fresh[i] : 0;
    if (in) {
      q_start[r] = at;
      len_s[r] = cached[i];
      base[r] = ok ? used : -1;
      if (blockIdx.x == 0) {
        a.q_start[r] = at;
        a.kv_len[r] = kv[i];
        a.next[r] = ok ? cached[i] + fresh[i] : cached[i];
      }
    }
    sums[4] += in && !ok && fresh[i] > 0;
    cnt[5] += in && ok ? n : 0;
    used += n;
    at += fresh[i];
    const int rows = min(fresh[i], a.row_limit) * a.group;
    const bool b = in_list_b(a, rows);
    tiles[i] = b ? (rows + a.s.rows_b - 1) / a.s.rows_b : rows > 0 ? -1 : 0;
    if (b) work += work_of(tiles[i], fresh[i], kv[i], a.s.rows_b, a.group);
    else if (rows > 0) sums[0] += pieces_of(kv[i]);
  }
  sums[1] = (int)(work & 0xFFFFF), sums[2] = (int)((work >> 20) & 0xFFFFF), sums[3] = (int)(work >> 40);
  block_scan<5, kThreads>(sums, sums_total, wsum, tid);
  work = sums_total[1] + ((long long)sums_total[2] << 20) + ((long long)sums_total[3] << 40);
  const int refused = sums_total[4];
  const int share = max(kLeastShare, (sums_total[0] + a.s.shares - 1) / a.s.shares);  // pieces
  // keys of work per CU: list b's tiles times keys, and half of list a's keys
  const float cu_keys = (float)(work + 32LL * sums_total[0]) / (float)max(a.s.target_b, 1);
  // units of each request: the shares that its pieces touch, or tiles of rows times parts of its keys
  int parts[kPer], split_tiles[kPer] = {}, split_parts[kPer] = {}, piece0[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    piece0[i] = sums[0];
    if (tiles[i] < 0) {
      const int end = sums[0] + pieces_of(kv[i]);
      parts[i] = (int)((unsigned)(end - 1) / (unsigned)share - (unsigned)sums[0] / (unsigned)share) + 1;
      sums[0] = end;
      cnt[0] += parts[i];
      cnt[3] += parts[i] > 1 ? parts[i] : 0;
    } else {
      if (a.s.target_b > 0 && tiles[i] > 0) {  // (there are fewer than 384 tiles then)
        const float per_key = parts_per_key(cu_keys, min(fresh[i], a.row_limit) * a.group, tiles[i], a.s.rows_b);
        for (int t = tiles[i] - 1; t >= 0; --t) {
          const int n = parts_of(tile_keys(t, fresh[i], kv[i], a.s.rows_b, a.group), per_key);
          if (n == 1) break;  // nor has a tile before it more
          ++split_tiles[i], split_parts[i] += n;
        }
      }
      parts[i] = tiles[i] - split_tiles[i] + split_parts[i];
      cnt[1] += parts[i], cnt[2] += split_tiles[i], cnt[4] += split_parts[i];
    }
  }
  int cnt_total[kPlanSums];
  block_scan<kPlanSums, kThreads>(cnt, cnt_total, wsum, tid);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = r0 + i;
    if (i >= per || r >= a.R) continue;
    if (tiles[i] < 0) {
      first[r] = cnt[0], split[r] = piece0[i], partial[r] = cnt[3];
      cnt[0] += parts[i];
      if (parts[i] > 1) cnt[3] += parts[i];
    } else {
      first[r] = cnt[1], split[r] = cnt[2], partial[r] = cnt[4];
      cnt[1] += parts[i], cnt[2] += split_tiles[i], cnt[4] += split_parts[i];
    }
  }
  if (tid == 0) q_start[a.R] = total[0];
  if (blockIdx.x == 0 && tid == 0) {
    a.q_start[a.R] = total[0];
    a.info[0] = (int)(((unsigned)head + (unsigned)cnt_total[5]) % N);
    a.info[1] = count - cnt_total[5];
    a.info[2] = refused;
    a.info[3] = total[0];
    a.sched[0] = min(cnt_total[0], a.s.max_units_a);
    a.sched[1] = min((sums_total[0] + share - 1) / share, a.s.shares);
    a.sched[2] = min(cnt_total[1], a.s.max_units_b);
    a.sched[3] = min(cnt_total[2], a.s.max_splits_b);
  }
  __syncthreads();
  // slots: one thread per token; a block's first token also writes its entry
  for (int t = (int)blockIdx.x * kThreads + tid; t < a.total; t += (int)gridDim.x * kThreads) {
    int lo = 0, hi = a.R;  // the last request with q_start <= t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (q_start[mid] <= t) lo = mid;
      else hi = mid;
    }
    long long slot = -1;
    // (lengths whose sum passes 32 bits leave q_start out of order: a token has a
    // slot only inside its request, whose blocks the table holds)
    if (t < q_start[a.R] && base[lo] >= 0 && (unsigned)t - (unsigned)q_start[lo] < (unsigned)q_start[lo + 1] - (unsigned)q_start[lo]) {
      const int c = len_s[lo];
      const int have = (c + a.B - 1) >> a.b_shift, p = c + t - q_start[lo], j = p >> a.b_shift;
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
  int32_t* shares = a.sched + a.s.off_shares;
  KvUnit* units_a = reinterpret_cast<KvUnit*>(a.sched + a.s.off_units_a);
  KvUnit* units_b = reinterpret_cast<KvUnit*>(a.sched + a.s.off_units_b);
  KvSplit* splits_b = reinterpret_cast<KvSplit*>(a.sched + a.s.off_splits_b);
  constexpr int kWaves = kThreads / kWave;
  for (int r = (int)blockIdx.x * kWaves + wave; r < a.R; r += (int)gridDim.x * kWaves) {
    const int q = q_start[r + 1] - q_start[r];
    if (q == 0) continue;
    const int len = base[r] >= 0 ? len_s[r] + q : 0;
    const int rows = min(q, a.row_limit) * a.group;
    KvUnit u = {};
    u.req = r;
    if (!in_list_b(a, rows)) {
      const int p0 = split[r], p1 = p0 + pieces_of(len), s0 = (int)((unsigned)p0 / (unsigned)share);
      const int n = (int)((unsigned)(p1 - 1) / (unsigned)share) - s0 + 1;
      for (int i = lane; i < n; i += kWave) {
        const int begin = max(p0, (s0 + i) * share), end = min(p1, (s0 + i + 1) * share), at = first[r] + i;
        u.row = 0;
        u.kv_begin = min((begin - p0) * 64, len);
        u.kv_end = min((end - p0) * 64, len);
        u.part = n > 1 ? partial[r] + i : -1;
        u.first = partial[r];
        u.parts = n;
        if ((unsigned)at < (unsigned)a.s.max_units_a && u.part < a.s.max_parts_a) units_a[at] = u;
        // every share starts with a unit of its own
        if (begin == (s0 + i) * share && s0 + i < a.s.shares) shares[s0 + i] = at;
      }
    } else {
      // a lane per tile; the last tile sees the most keys: it goes first
      const int tiles_r = (rows + a.s.rows_b - 1) / a.s.rows_b;
      int at = first[r], part = partial[r], join = split[r];
      if (a.s.target_b == 0) {  // no tile is split
        u.part = -1;
        for (int i = lane; i < tiles_r; i += kWave) {
          const int tile = tiles_r - 1 - i;
          u.row = tile * a.s.rows_b;
          u.kv_end = tile_keys(tile, q, len, a.s.rows_b, a.group);
          if ((unsigned)(at + i) < (unsigned)a.s.max_units_b) units_b[at + i] = u;
        }
        continue;
      }
      const float per_key = parts_per_key(cu_keys, rows, tiles_r, a.s.rows_b);
      for (int i0 = 0; i0 < tiles_r; i0 += kWave) {
        const int tile = tiles_r - 1 - i0 - lane;
        const int seen = tile >= 0 ? tile_keys(tile, q, len, a.s.rows_b, a.group) : 0;
        const int n = tile < 0 ? 0 : parts_of(seen, per_key), m = n > 1 ? n : 0;
        const int n_sum = wave_scan(n), m_sum = wave_scan(m);
        const unsigned long long splits = __ballot(m > 0);
        const int my_at = at + n_sum - n, my_part = part + m_sum - m;
        const int each = n <= 1 ? seen : ((int)((unsigned)(seen + n - 1) / (unsigned)n) + 63) & ~63;
        u.row = tile * a.s.rows_b;
        for (int p = 0; p < n; ++p) {
          u.kv_begin = min(p * each, seen);
          u.kv_end = min((p + 1) * each, seen);
          u.part = n > 1 ? my_part + p : -1;
          if ((unsigned)(my_at + p) < (unsigned)a.s.max_units_b && u.part < a.s.max_parts_b) units_b[my_at + p] = u;
        }
        const int my_join = join + __popcll(splits & ((1ull << lane) - 1));
        if (m > 0 && (unsigned)my_join < (unsigned)a.s.max_splits_b) splits_b[my_join] = KvSplit{r, u.row, my_part, n};
        at += __builtin_amdgcn_readlane(n_sum, kWave - 1), part += __builtin_amdgcn_readlane(m_sum, kWave - 1);
        join += __popcll(splits);
      }
    }
  }
}

constexpr int kPlanThreads = 1024;

// Lengths, ring state and (for finished requests) the table after a step.  A
// finished request's blocks return to the ring's end in the order of requests
// and of their tables.  One workgroup, as lengths and state are read and
// written in place; a running sum of the finished requests' blocks in LDS gives
// every entry a thread of its own (with a thread per request the end of one of
// 8192 blocks took 1100 us, now 10).
__global__ void __launch_bounds__(kPlanThreads) k_kv_commit(KvCommitArgs a) {
  __shared__ int wsum[1][16];
  __shared__ int before[kKvMaxRequests];  // entries of finished requests before this one
  const int tid = threadIdx.x;
  const int per = (a.R + kPlanThreads - 1) / kPlanThreads, r0 = tid * per;
  const unsigned N = (unsigned)a.num_blocks;
  const int* from = a.info != nullptr ? a.info : a.state;
  const int head = (int)((unsigned)from[0] % N), count = min(max(from[1], 0), a.num_blocks);
  const auto length = [&](int r) { return clip_len(a.next != nullptr ? a.next[r] : a.cached[r]); };
  int mine[1] = {0}, total[1] = {0};
  if (a.finished != nullptr) {
    for (int i = 0; i < per && r0 + i < a.R; ++i) {
      before[r0 + i] = mine[0];
      if (a.finished[r0 + i] != 0) mine[0] += min((length(r0 + i) + a.B - 1) >> a.b_shift, a.max_blocks);
    }
    block_scan<1, kPlanThreads>(mine, total, wsum, tid);
    for (int i = 0; i < per && r0 + i < a.R; ++i) before[r0 + i] += mine[0];
  }
  __syncthreads();
  for (int e = tid; e < total[0]; e += kPlanThreads) {
    int lo = 0, hi = a.R;  // the last request with before <= e
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= e) lo = mid;
      else hi = mid;
    }
    int32_t* entry = a.table + (long long)lo * a.max_blocks + (e - before[lo]);
    // never more than the ring holds: a table with an id twice cannot push the ring past its size
    if (count + e < a.num_blocks) a.ring[((unsigned)head + (unsigned)(count + e)) % N] = *entry;
    *entry = -1;
  }
  for (int i = 0; i < per && r0 + i < a.R; ++i) {
    const int r = r0 + i;
    if (a.finished != nullptr && a.finished[r] != 0) a.cached[r] = 0;
    else if (a.next != nullptr) a.cached[r] = a.next[r];
  }
  if (tid == 0) {
    a.state[0] = head;
    a.state[1] = min(count + total[0], a.num_blocks);
  }
}

// ---------------------------------------------------------------- append --
// One wave per (run, head, K or V): a run is the tokens of one block, which
// stand next to each other in the call.  A wave looks at kTake tokens for the
// first of a run; where there are few tokens it takes one.  A run's rows are
// loaded once, all loads in flight together, and stay in registers between the
// search for the largest magnitude and the coding.
//
// K: a lane holds 16 dims of a token (16 code bytes).  V: a lane holds 4 dims
// of 4 tokens, which is how V's codes lie; the wave owns the block's V, so
// bytes of other tokens in a piece of 16 are read and written back.
//
// What bounds it: memory latency.  A run is slots, rows, scale, codes one after
// the other: 64 single tokens of 8 heads 4.1 us, next to an empty launch's 2.4;
// 11420 tokens of prompts (70 MB) 21 us, 3.3 TB/s.
constexpr int kAppendThreads = 256;

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

// Codes of four values under scale s (r = 1 / s rounded), in byte order.  The
// int8 quotient is rounded as a division: x r corrected by its residual (a
// correctly rounded r makes the corrected product the correctly rounded
// quotient); adding 1.5 2^23 + 128 rounds it to an integer, to even, and leaves
// code + 128 in the low byte (|x / s| < 127.5, as s is at least the largest
// magnitude / 127).  An e4m3 scale is a power of two: x r is exact.  Under a NaN
// scale e4m3 codes are zero: the scale makes their values NaN, and a NaN code
// would also reach rows of the attention that give it a weight of zero.
template <int kFmt>
__device__ __forceinline__ uint32_t kv_encode4(const float (&x)[4], float s, float r) {
  if constexpr (kFmt == NSMLP_KV_INT8) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float q = x[i] * r;
      const float y = __builtin_fmaf(__builtin_fmaf(-q, s, x[i]), r, q);
      c[i] = __float_as_uint(y + 12583040.0f);
    }
    const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000C0Cu);
    return lo | hi;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * r, x[1] * r, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * r, x[3] * r, w, true);
    return s == s ? (uint32_t)w : 0u;
  }
}

// A stored dword's codes under a larger scale.
template <int kFmt>
__device__ __forceinline__ uint32_t kv_recode4(uint32_t w, float s_old, float s, float r) {
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = kv_decode1<kFmt>((w >> (8 * i)) & 0xFFu) * s_old;
  return kv_encode4<kFmt>(x, s, r);
}

__device__ __forceinline__ uint32_t top16(uint32_t top, uint32_t w) {
  return max(top, max(w & 0x7FFFu, (w >> 16) & 0x7FFFu));
}

template <int D, int B, int kFmt, bool kBf16>
__device__ __forceinline__ void append_run(const KvAppendArgs& a, int t, long long slot, int n, int h, bool is_v, int lane) {
  const long long blk = slot / B;
  const int o0 = (int)(slot & (B - 1));  // first new offset
  float* sp = a.c.scale + (blk * a.c.heads + h) * 2 + (is_v ? 1 : 0);
  uint8_t* dst = a.c.data + ((blk * a.c.heads + h) * 2 + (is_v ? 1 : 0)) * (long long)(B * D);
  const float s_old = o0 == 0 ? 0.0f : *sp;
  const auto settle = [&](uint32_t top, float& s, float& r, bool& recode) {
    // largest magnitude, as bits (a NaN or infinity is above every finite value)
#pragma unroll
    for (int m = kWave / 2; m >= 1; m >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m, kWave));
    const float need = kv_scale_of<kFmt>(in_value<kBf16>(top));
    // a NaN on either side stays until the block is started anew
    s = need != need || s_old != s_old ? __uint_as_float(0x7FC00000u) : fmaxf(s_old, need);
    r = 1.0f / s;
    recode = o0 > 0 && s != s_old;
    if (lane == 0) *sp = s;
  };
  float s, r;
  bool recode;
  if (!is_v) {
    constexpr int kChunks = D / 16, kTok = kWave / kChunks, kPass = B / kTok;  // tokens of a pass
    const int tl = lane / kChunks, c = lane % kChunks;
    const uint16_t* x = a.k + (long long)t * a.k_row + (long long)h * a.k_head + c * 16;
    uint4 u[kPass][2];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
      const int i = p * kTok + tl;
      u[p][0] = u[p][1] = uint4{0, 0, 0, 0};
      if (i < n) {
        const uint4* q = reinterpret_cast<const uint4*>(x + i * a.k_row);
        u[p][0] = q[0], u[p][1] = q[1];
      }
    }
#pragma unroll
    for (int p = 0; p < kPass; ++p)
#pragma unroll
      for (int j = 0; j < 2; ++j) top = top16(top16(top16(top16(top, u[p][j].x), u[p][j].y), u[p][j].z), u[p][j].w);
    settle(top, s, r, recode);
    if (recode) {
      for (int i = tl; i < o0; i += kTok) {
        uint4* q = reinterpret_cast<uint4*>(dst + kv_k_off(D, i, c * 16));
        const uint4 w = *q;
        *q = uint4{kv_recode4<kFmt>(w.x, s_old, s, r), kv_recode4<kFmt>(w.y, s_old, s, r), kv_recode4<kFmt>(w.z, s_old, s, r),
                   kv_recode4<kFmt>(w.w, s_old, s, r)};
      }
    }
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
      const int i = p * kTok + tl;
      if (i < n) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4& v = u[p][j >> 1];
          const uint32_t w0 = j & 1 ? v.z : v.x, w1 = j & 1 ? v.w : v.y;
          const float e[4] = {in_lo<kBf16>(w0), in_hi<kBf16>(w0), in_lo<kBf16>(w1), in_hi<kBf16>(w1)};
          o[j] = kv_encode4<kFmt>(e, s, r);
        }
        *reinterpret_cast<uint4*>(dst + kv_k_off(D, o0 + i, c * 16)) = uint4{o[0], o[1], o[2], o[3]};
      }
    }
  } else {
    constexpr int kPieces = D / 4, kGroups = kWave / kPieces, kPass = B / 4 / kGroups;
    const int gl = lane / kPieces, d0 = lane % kPieces * 4;
    const uint16_t* x = a.v + ((long long)t - o0) * a.v_row + (long long)h * a.v_head + d0;
    uint2 u[kPass][4];
    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < kPass; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int off = 4 * (p * kGroups + gl) + i;
        u[p][i] = uint2{0, 0};
        if (off >= o0 && off < o0 + n) u[p][i] = *reinterpret_cast<const uint2*>(x + off * a.v_row);
      }
#pragma unroll
    for (int p = 0; p < kPass; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = top16(top16(top, u[p][i].x), u[p][i].y);
    settle(top, s, r, recode);
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
      const int first = 4 * (p * kGroups + gl);
      if (first >= o0 + n || (!recode && first + 4 <= o0)) continue;
      uint4* q = reinterpret_cast<uint4*>(dst + kv_v_off(D, first, d0));
      // bytes of tokens before, in and after the run
      const int lo = min(max(o0 - first, 0), 4), hi = min(o0 + n - first, 4);
      const uint32_t before = lo == 4 ? ~0u : (1u << (8 * lo)) - 1u, upto = hi == 4 ? ~0u : (1u << (8 * hi)) - 1u;
      uint4 old = uint4{0, 0, 0, 0};
      if (lo > 0 || hi < 4) old = *q;
      const uint32_t w[4] = {old.x, old.y, old.z, old.w};
      uint32_t o[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t v = d < 2 ? u[p][i].x : u[p][i].y;
          e[i] = d & 1 ? in_hi<kBf16>(v) : in_lo<kBf16>(v);
        }
        const uint32_t kept = recode && lo > 0 ? kv_recode4<kFmt>(w[d], s_old, s, r) : w[d];
        o[d] = (kept & before) | (kv_encode4<kFmt>(e, s, r) & upto & ~before) | (w[d] & ~upto);
      }
      *q = uint4{o[0], o[1], o[2], o[3]};
    }
  }
}

template <int D, int B, int kFmt, bool kBf16>
__global__ void __launch_bounds__(kAppendThreads, B == 64 ? 2 : 4) k_kv_append(KvAppendArgs a) {
  kernarg_warm<sizeof(KvAppendArgs)>();
  const int lane = threadIdx.x & (kWave - 1);
  const int item = (int)blockIdx.x * (kAppendThreads / kWave) + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int two_heads = 2 * a.c.heads;
  const int t0 = item / two_heads * a.take, hk = item % two_heads;
  if (t0 >= a.n) return;
  const long long limit = (long long)a.c.num_blocks * B;
  // Slots of the wave's tokens and of the 64 after them, in one round trip:
  // which start a run, and which go on with the one before them.
  const auto slot_at = [&](int t) -> long long {
    const long long v = t >= 0 && t < a.n ? a.slots[t] : -1;
    return v < limit ? v : -1;
  };
  const long long s0 = slot_at(t0 + lane), s1 = slot_at(t0 + kWave + lane), p0 = slot_at(t0 + lane - 1), p1 = slot_at(t0 + kWave + lane - 1);
  const bool on0 = s0 >= 0 && p0 == s0 - 1 && (s0 & (B - 1)) != 0, on1 = s1 >= 0 && p1 == s1 - 1 && (s1 & (B - 1)) != 0;
  const unsigned long long go0 = __ballot(on0), go1 = __ballot(on1);
  unsigned long long todo = __ballot(lane < a.take && s0 >= 0 && !on0);
  while (todo != 0) {
    const int i = __builtin_ctzll(todo);
    todo &= todo - 1;
    // tokens i + 1 ... that go on: at most B - 1 <= 63 of them
    const unsigned long long after = i == kWave - 1 ? go1 : (go0 >> (i + 1)) | (go1 << (kWave - 1 - i));
    const int n = after == ~0ull ? kWave : 1 + __builtin_ctzll(~after);
    const long long slot = ((long long)__builtin_amdgcn_readlane((int)(s0 >> 32), i) << 32) |
                           (uint32_t)__builtin_amdgcn_readlane((int)s0, i);
    append_run<D, B, kFmt, kBf16>(a, t0 + i, slot, min(n, B - (int)(slot & (B - 1))), hk >> 1, hk & 1, lane);
  }
}

// ------------------------------------------------------------------ read --
// One thread per 16 dims of a (slot, head): values code * scale, rounded once.
// The token's V bytes lie one in each dword of 4 pieces of 16; the threads of
// the group's other tokens find the same pieces in the caches.  11532 tokens of
// 8 heads (71 MB) 17-18 us, 4 TB/s, three quarters of what a copy reaches.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
  if constexpr (kBf16) return __builtin_bit_cast(uint16_t, (__bf16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)b) << 16;
  else return f2h(a) | (uint32_t)f2h(b) << 16;
}

template <int D, int kFmt, bool kBf16>
__global__ void __launch_bounds__(256) k_kv_read(KvReadArgs a) {
  kernarg_warm<sizeof(KvReadArgs)>();
  constexpr int kPer = D / 16;
  const unsigned item = blockIdx.x * 256u + threadIdx.x;
  const int c = (int)(item % kPer);
  const unsigned th = item / kPer;
  const int h = (int)(th % (unsigned)a.c.heads);
  const int t = (int)(th / (unsigned)a.c.heads);
  if (t >= a.n) return;
  const long long slot = a.slots[t];
  uint32_t ko[8] = {}, vo[8] = {};
  if (slot >= 0 && slot < (long long)a.c.num_blocks * a.c.B) {
    const long long bh = (slot >> a.c.b_shift) * a.c.heads + h;
    const int off = (int)(slot & (a.c.B - 1)), sh = 8 * (off & 3);
    const uint8_t* kb = a.c.data + bh * 2 * (long long)(a.c.B * D);
    const uint4 kw = *reinterpret_cast<const uint4*>(kb + kv_k_off(D, off, c * 16));
    const uint4* vp = reinterpret_cast<const uint4*>(kb + a.c.B * D + kv_v_off(D, off & ~3, c * 16));
    const uint4 vw[4] = {vp[0], vp[1], vp[2], vp[3]};
    const float2 s = *reinterpret_cast<const float2*>(a.c.scale + bh * 2);
    const uint32_t kd[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float k[4], v[4];
      const uint32_t vd[4] = {vw[j].x, vw[j].y, vw[j].z, vw[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k[i] = kv_decode1<kFmt>((kd[j] >> (8 * i)) & 0xFFu) * s.x;
        v[i] = kv_decode1<kFmt>((vd[i] >> sh) & 0xFFu) * s.y;
      }
      ko[2 * j] = pack_out<kBf16>(k[0], k[1]), ko[2 * j + 1] = pack_out<kBf16>(k[2], k[3]);
      vo[2 * j] = pack_out<kBf16>(v[0], v[1]), vo[2 * j + 1] = pack_out<kBf16>(v[2], v[3]);
    }
  }
  const long long o = ((long long)t * a.c.heads + h) * D + c * 16;
  uint4 *kp = reinterpret_cast<uint4*>(a.k + o), *vp = reinterpret_cast<uint4*>(a.v + o);
  kp[0] = uint4{ko[0], ko[1], ko[2], ko[3]}, kp[1] = uint4{ko[4], ko[5], ko[6], ko[7]};
  vp[0] = uint4{vo[0], vo[1], vo[2], vo[3]}, vp[1] = uint4{vo[4], vo[5], vo[6], vo[7]};
}

template <int D, int kFmt, bool kBf16>
void append_typed(KvAppendArgs a, hipStream_t s) {
  // Most tokens of a long call are a prompt's, and the waves that find no first
  // token of a run cost a round trip each: several tokens per wave where even
  // then every CU has a dozen waves.  Single tokens that stand next to each other
  // are then one wave's, one after the other.  With 1, 8 and 16 tokens per wave,
  // 8 heads: prompts of 4096 tokens (65536 pairs) 32.6, 10.5, 9.6 us, of 8192 62.5,
  // 17.0, 13.9; single tokens, 1024 of them 16.0, 17.7, 28.2 us, 2048 29.0, 23.0, 32.1,
  // 4096 53.9, 41.1, 41.7; 290 next to 7000 of prompts 46.9, 18.3, 30.2.
  const long long pairs = (long long)a.n * a.c.heads * 2;
  a.take = pairs >= 128 * 1024 ? 16 : pairs >= 32 * 1024 ? 8 : 1;
  const long long waves = (long long)((a.n + a.take - 1) / a.take) * a.c.heads * 2, per = kAppendThreads / kWave;
  const dim3 grid((unsigned)((waves + per - 1) / per)), block(kAppendThreads);
  if (a.c.B == 16) k_kv_append<D, 16, kFmt, kBf16><<<grid, block, 0, s>>>(a);
  else if (a.c.B == 32) k_kv_append<D, 32, kFmt, kBf16><<<grid, block, 0, s>>>(a);
  else k_kv_append<D, 64, kFmt, kBf16><<<grid, block, 0, s>>>(a);
}

template <int D, int kFmt, bool kBf16>
void read_typed(const KvReadArgs& a, hipStream_t s) {
  const long long items = (long long)a.n * a.c.heads * (D / 16);
  k_kv_read<D, kFmt, kBf16><<<dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s>>>(a);
}

}  // namespace

void launch_kv_append(const KvAppendArgs& a, bool bf16, hipStream_t s) { NSMLP_KV_BY_TYPE(append_typed, a, bf16, s); }
void launch_kv_read(const KvReadArgs& a, bool bf16, hipStream_t s) { NSMLP_KV_BY_TYPE(read_typed, a, bf16, s); }

KvSchedule kv_schedule(int requests, int total, int max_new, int group, int kv_heads) {
  KvSchedule s;
  // list a: one workgroup of 4 waves per CU has as many reads in flight as the
  // memory takes (two: 131000 keys 57.9 -> 62.5 us, for the joins)
  s.shares = (256 + kv_heads - 1) / kv_heads;
  // list b: 256 rows per workgroup where that still makes two for every CU
  // (chunk of 2048 over 14336, 128 heads: 2.01 ms, with 128 rows 2.11), else 128
  const long long rows = (long long)total * group;
  s.rows_b = rows / 256 * kv_heads >= 512 ? 256 : 128;
  const long long most = (long long)(max_new < total ? max_new : total) * group;
  s.list_b = most > kKvRowsA;
  s.join_rows = most < s.rows_b ? (int)most : s.rows_b;
  const long long tiles_b = s.list_b ? (rows + s.rows_b - 1) / s.rows_b + requests : 0;
  // its keys are shared out where the tiles do not make one and a half for every CU
  s.target_b = !s.list_b || tiles_b * kv_heads >= 384 ? 0 : (256 + kv_heads - 1) / kv_heads;
  // list a: every share ends at most one unit that its request does not end,
  // so units are at most requests + shares, and those of a request with several
  // units at most twice the shares
  s.max_units_a = requests + s.shares;
  s.max_parts_a = 2 * s.shares;
  // list b: a tile has two parts or more only past 1.35 L keys, and L is at least
  // half the work over the target: split tiles are below 1.5 targets, their parts below 3
  s.max_parts_b = 3 * s.target_b;
  s.max_splits_b = 2 * s.target_b;
  s.max_units_b = (int)tiles_b + s.max_parts_b;
  const long long unit = sizeof(KvUnit) / 4, split = sizeof(KvSplit) / 4;
  s.off_shares = kKvHeaderInts;
  s.off_units_a = s.off_shares + (s.shares + 3) / 4 * 4;
  s.off_units_b = s.off_units_a + unit * s.max_units_a;
  s.off_splits_b = s.off_units_b + unit * s.max_units_b;
  s.ints = s.off_splits_b + split * s.max_splits_b;
  return s;
}

template <int kThreads, int kPer>
static void launch_plan(const KvPlanArgs& a, hipStream_t s) {
  static std::once_flag once;
  constexpr int kMost = (6 * kThreads * kPer + 1) * (int)sizeof(int);
  std::call_once(once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(k_kv_plan<kThreads, kPer>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
  });
  // two tokens per thread and 16 requests' lists per workgroup, but one workgroup per
  // CU at most (64 requests' lists and 128 workgroups: 4096 requests 17 us, now 14)
  const int groups = min(max((a.total + 2 * kThreads - 1) / (2 * kThreads), (a.R + 15) / 16), 256);
  k_kv_plan<kThreads, kPer><<<dim3(max(groups, 1)), dim3(kThreads), (6 * a.R + 1) * sizeof(int), s>>>(a);
}

void launch_kv_plan(const KvPlanArgs& a, hipStream_t s) {
  if (a.R <= 64) launch_plan<64, 1>(a, s);
  else if (a.R <= 256) launch_plan<256, 1>(a, s);
  else if (a.R <= 1024) launch_plan<1024, 1>(a, s);
  else launch_plan<1024, kKvMaxRequests / 1024>(a, s);
}

void launch_kv_commit(const KvCommitArgs& a, hipStream_t s) {
  k_kv_commit<<<dim3(1), dim3(kPlanThreads), 0, s>>>(a);
}

}  // namespace nsmlp
