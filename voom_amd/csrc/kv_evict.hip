// Eviction from a paged K/V cache by accumulated attention weight, for gfx950: which
// tokens of each head stay (evict_select_kernel), and the move of the rows that stay
// to the front (compact_kernel, which also keeps the accepted branch of a tree of
// drafts).
#include "common.h"

namespace voom {
namespace {

// ---- selection -----------------------------------------------------------------
//
// Of a (sequence, kv head) with ctx > budget tokens stay the first `sink`, the newest
// `recent`, and of those between the n = budget - sink - recent of largest score, equal
// ones lowest position first.  Scores are ordered as integers (a NaN lowest of all,
// -0 as 0); three histogram passes over 11, 11 and 10 bits find the n-th largest one,
// and a last pass writes the positions in ascending order.
//
// What bounds it: the scores once, 4 bytes per token and head, and the latency of one
// workgroup per (sequence, head).  Up to 32,768 candidates stay in registers, all loads
// in flight at once (a loop that loaded them for every pass: 43 us for 16 x 8 heads of
// up to 32,768 tokens, where this takes 17); of longer ones every pass loads 32,768 at a
// time (64 heads of 131,072: 58 us; 65 before the lists had one atomic a wavefront, and with
// 49,152 at a time, some of them spilled, 76).
// Each histogram of a long row has eight copies, by lane: scores share their leading
// bits, and atomics of one wavefront on one address take turns.  The second and third
// pass look only at the keys that share the first digit, from a list in LDS where it
// holds them.

constexpr int kBins = 2048;
constexpr int kList = 16384;  // candidates that share their first digit with the n-th largest

// Larger score, larger key; NaN 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 + 0 is 0
  const uint32_t k = (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
  return x != x ? 0u : k;
}

// Exclusive prefix sum of the wavefronts' totals (at most 16) for wavefront wv, and
// their sum.
template <int WAVES>
__device__ __forceinline__ int before_wave(const int* tot, int wv, int lane, int& all) {
  const int x = wave_inclusive_scan(lane < WAVES ? tot[lane] : 0, lane);
  all = __builtin_amdgcn_readlane(x, kWave - 1);
  return wv == 0 ? 0 : __builtin_amdgcn_readlane(x, wv - 1);
}

// Which bin of a histogram holds the need-th largest key.  Thread t holds, in `mine`, bins
// t per .. of the descending order, per = bins / THREADS.
template <int THREADS>
__device__ __forceinline__ void find_digit(const int (&mine)[kBins / THREADS], int bins, int need,
                                           int* part, int* found) {
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & (kWave - 1);
  const int wv = uniform(tid / kWave);
  constexpr int kPer = kBins / THREADS;
  const int per = bins / THREADS;
  int sum = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) sum += mine[j];
  const int x = wave_inclusive_scan(sum, lane);
  if (lane == kWave - 1) part[wv] = x;
  __syncthreads();
  int all;
  int before = before_wave<THREADS / kWave>(part, wv, lane, all) + x - sum;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (j < per && before < need && before + mine[j] >= need) {
      found[0] = bins - 1 - (tid * per + j);
      found[1] = before;
      found[2] = mine[j];
    }
    before += mine[j];
  }
  __syncthreads();
}

// Writes the positions of the candidates in registers that stay: of those equal to
// `prefix`, the n-th largest key, the first `need`, mostly all of them (all_equal).  Each
// wavefront counts what its run of the candidates keeps, and writes behind the runs before
// it; at, same: how many were kept, and (where not all stay) equal to the key, before.
template <int THREADS, int E>
__device__ __forceinline__ void write_kept(uint32_t (&key)[E], int first, int count,
                                           uint32_t prefix, int need, bool all_equal, int sink,
                                           int32_t* out, int* kept_tot, int* equal_tot, int& at,
                                           int& same) {
  constexpr int kWaves = THREADS / kWave;
  const int lane = static_cast<int>(threadIdx.x) & (kWave - 1);
  const int wv = uniform(static_cast<int>(threadIdx.x) / kWave);
  int kept = 0, equal = 0;
  if (all_equal) {
#pragma unroll
    for (int e = 0; e < E; ++e) kept += __popcll(__builtin_amdgcn_ballot_w64(key[e] >= prefix));
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      kept += __popcll(__builtin_amdgcn_ballot_w64(key[e] > prefix));
      equal +=
          __popcll(__builtin_amdgcn_ballot_w64(key[e] == prefix && first + e * kWave < count));
    }
  }
  // (keeps the compiler from holding two lane masks per element until below)
#pragma unroll
  for (int e = 0; e < E; ++e) asm volatile("" : "+v"(key[e]));
  __syncthreads();  // the totals of the call before are read
  if (lane == 0) {
    kept_tot[wv] = kept;
    equal_tot[wv] = equal;
  }
  __syncthreads();
  int kept_all, equal_all;
  int run_at = at + before_wave<kWaves>(kept_tot, wv, lane, kept_all);
  int run_same = same + before_wave<kWaves>(equal_tot, wv, lane, equal_all);
  at += kept_all;
  same += equal_all;
  if (all_equal) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t up = __builtin_amdgcn_ballot_w64(key[e] >= prefix);
      if (key[e] >= prefix)
        out[sink + run_at +
            __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(up >> 32),
                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(up), 0))] =
            sink + first + e * kWave;
      run_at += __popcll(up);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool same_key = key[e] == prefix && first + e * kWave < count;
      const uint64_t up = __builtin_amdgcn_ballot_w64(key[e] > prefix);
      const uint64_t eq = __builtin_amdgcn_ballot_w64(same_key);
      const uint64_t low = (1ull << lane) - 1;
      const int eq_before = run_same + __popcll(eq & low);
      if (key[e] > prefix || (same_key && eq_before < need)) {
        const int eq_kept = eq_before < need ? eq_before : need;
        out[sink + run_at + __popcll(up & low) + eq_kept] = sink + first + e * kWave;
      }
      run_at += __popcll(up);
      run_same += __popcll(eq);
    }
  }
}

// This thread's keys of the candidates from `first` on, 64 apart, 0 past the last one.
template <int E>
__device__ __forceinline__ void load_keys(const float* s, int first, int count,
                                          uint32_t (&key)[E]) {
  // (candidates past the last one load 0: the whole offset is in the part of the address
  // that is checked)
  const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<float*>(s), static_cast<short>(0), count * 4u, 0x00020000);
#pragma unroll
  for (int e = 0; e < E; ++e)
    key[e] = __builtin_amdgcn_raw_buffer_load_b32(from, (first + e * kWave) * 4u, 0, 0);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t k = order_key(__builtin_bit_cast(float, key[e]));
    key[e] = first + e * kWave < count ? k : 0u;
  }
}

// The digits of a key from the highest on, 11, 11 and 10 bits.
__device__ __forceinline__ int digit_shift(int pass) {
  return pass == 0 ? 21 : (pass == 1 ? 10 : 0);
}
__device__ __forceinline__ int digit_bins(int pass) { return pass == 2 ? 1024 : 2048; }

// E: candidates per thread and round.  Round c, wavefront w, element e, lane l hold
// candidate ((c * waves + w) * E + e) * 64 + l; past the last one the key is 0.
// COPIES: of the histogram, by lane.
template <int kSelThreads, int E, int COPIES>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(
    const float* __restrict__ scores, const int32_t* __restrict__ ctx_lens,
    int32_t* __restrict__ keep, int32_t* __restrict__ keep_lens, int NKV, int cap, int budget,
    int sink, int recent) {
  constexpr int kSelWaves = kSelThreads / kWave;
  __shared__ __attribute__((aligned(16))) int hist[kBins][COPIES];
  __shared__ uint32_t list[E > 8 ? kList : 1];
  __shared__ int listed;
  __shared__ int part[kSelWaves];
  __shared__ int found[3];  // digit that holds the n-th largest; keys above it, keys in it
  __shared__ int kept_tot[kSelWaves], equal_tot[kSelWaves];
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & (kWave - 1);
  const int wv = uniform(tid / kWave);
  const int row = static_cast<int>(blockIdx.x);
  const int b = row / NKV;
  int ctx = uniform(ctx_lens[b]);
  ctx = ctx < 0 ? 0 : (ctx > cap ? cap : ctx);
  int32_t* out = keep + static_cast<size_t>(row) * budget;
  if (row == b * NKV && tid == 0) keep_lens[b] = ctx < budget ? ctx : budget;
  if (ctx <= budget) {
    for (int i = tid; i < budget; i += kSelThreads) out[i] = i < ctx ? i : -1;
    return;
  }
  const int n = budget - sink - recent;
  const float* s = scores + static_cast<size_t>(row) * cap + sink;
  const int count = ctx - recent - sink;  // candidates, more than n
  const int rounds = (count + kSelThreads * E - 1) / (kSelThreads * E);

  uint32_t key[E];
  auto first_of = [&](int c) { return (c * kSelWaves + wv) * (E * kWave) + lane; };
  auto load = [&](int c) { load_keys<E>(s, first_of(c), count, key); };
  if (n != 0) load(0);
  for (int i = tid; i < sink; i += kSelThreads) out[i] = i;
  for (int i = tid; i < recent; i += kSelThreads) out[budget - recent + i] = ctx - recent + i;
  if (n == 0) return;

  uint32_t prefix = 0, mask = 0;  // the bits of the n-th largest key found so far
  int need = n;                   // its rank among the keys with that prefix
  bool short_list = false;        // those keys are in `list`
  if (tid == 0) listed = 0;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = digit_shift(pass), bins = digit_bins(pass);
    int* const flat = &hist[0][0];  // one copy serves a short list
    const int cells = short_list ? bins : kBins * COPIES;
    for (int i = tid; i < cells / 4; i += kSelThreads)
      reinterpret_cast<u32x4*>(flat)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    if (short_list) {
      for (int i = tid; i < listed; i += kSelThreads)
        if ((list[i] & mask) == prefix) atomicAdd(&flat[(list[i] >> shift) & (bins - 1)], 1);
    } else {
      for (int c = 0; c < rounds; ++c) {
        if (rounds > 1 && (pass > 0 || c > 0)) load(c);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (first_of(c) + e * kWave < count && (key[e] & mask) == prefix)
            atomicAdd(&hist[(key[e] >> shift) & (bins - 1)][lane % COPIES], 1);
        }
      }
    }
    __syncthreads();
    // thread t owns bins t * per .. of the descending order
    constexpr int kPer = kBins / kSelThreads;
    const int per = bins / kSelThreads;
    int mine[kPer] = {};
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int bin = bins - 1 - (tid * per + j);
      if (j < per) {
        if (short_list) {
          mine[j] = flat[bin];
        } else {
#pragma unroll
          for (int k = 0; k < COPIES; ++k) mine[j] += hist[bin][k];
        }
      }
    }
    find_digit<kSelThreads>(mine, bins, need, part, found);
    prefix |= static_cast<uint32_t>(found[0]) << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    need -= found[1];
    if (E > 8 && pass == 0 && found[2] <= kList) {
      short_list = true;
      for (int c = 0; c < rounds; ++c) {
        if (rounds > 1) load(c);
        // (one atomic a wavefront: each waits for its answer)
        int mine_here = 0;
#pragma unroll
        for (int e = 0; e < E; ++e)
          mine_here += first_of(c) + e * kWave < count && (key[e] & mask) == prefix ? 1 : 0;
        const int x = wave_inclusive_scan(mine_here, lane);
        int at = 0;
        if (lane == kWave - 1) at = atomicAdd(&listed, x);
        at = __builtin_amdgcn_readlane(at, kWave - 1) + x - mine_here;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (first_of(c) + e * kWave < count && (key[e] & mask) == prefix) list[at++] = key[e];
      }
    }
  }

  const bool all_equal = prefix != 0 && need == found[2];
  int at = 0, same = 0;
  for (int c = 0; c < rounds; ++c) {
    if (rounds > 1) load(c);
    write_kept<kSelThreads, E>(key, first_of(c), count, prefix, need, all_equal, sink, out,
                               kept_tot, equal_tot, at, same);
  }
}

// Few rows of more than kRowMost scores: a workgroup takes a piece of kPiece candidates,
// and the row goes through four launches.  Pass 0, 1 and 2 count a digit of the piece's
// keys, and pass 1, 2 and 3 find the one before from all pieces' counts; pass 3 writes,
// behind what the pieces before it keep.  8 rows of 131,072: 28 us, 57 for one workgroup per
// row; 64 rows: 54 and 58; 128 rows of 65,536, which fill the card by themselves, 46 and 33;
// 8 rows of 36,000: 22 and 31.
constexpr int kSplitThreads = 1024;
constexpr int kSplitE = 16;
constexpr int kPiece = kSplitThreads * kSplitE;
constexpr int kRowMost = 32 * 1024;
constexpr int kMostPieces = 64;  // (each workgroup adds up the counts of all)
constexpr int kFewSplit = 64;    // rows

// A row's part of the workspace.
struct SplitRow {
  int* hist;   // [3][pieces][kBins]
  int* above;  // [2][pieces]: a piece's keys above the digit, of those that share the digits before
  int* found;  // [2][2]: the digit, and how many keys of the row lie above it
  __device__ __forceinline__ SplitRow(int* ws, int row, int pieces) {
    hist = ws + static_cast<size_t>(row) * ints(pieces);
    above = hist + 3 * pieces * kBins;
    found = above + 2 * pieces;
  }
  __host__ __device__ static constexpr size_t ints(int pieces) {
    return static_cast<size_t>(3) * pieces * kBins + 2 * pieces + 4;
  }
};

template <int PASS>
__global__ __launch_bounds__(kSplitThreads) void evict_split_kernel(
    const float* __restrict__ scores, const int32_t* __restrict__ ctx_lens,
    int32_t* __restrict__ keep, int32_t* __restrict__ keep_lens, int* __restrict__ ws, int NKV,
    int cap, int budget, int sink, int recent, int pieces) {
  constexpr int kWaves = kSplitThreads / kWave, kCopies = 8;
  __shared__ __attribute__((aligned(16))) int hist[PASS < 3 ? kBins : 1][kCopies];
  __shared__ int part[kWaves], kept_tot[kWaves], equal_tot[kWaves];
  __shared__ int found[3];
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & (kWave - 1);
  const int wv = uniform(tid / kWave);
  const int piece = static_cast<int>(blockIdx.x);
  const int row = static_cast<int>(blockIdx.y);
  const int b = row / NKV;
  int ctx = uniform(ctx_lens[b]);
  ctx = ctx < 0 ? 0 : (ctx > cap ? cap : ctx);
  int32_t* out = keep + static_cast<size_t>(row) * budget;
  const int n = budget - sink - recent;
  if (PASS == 0) {  // what needs no choice
    const int at = piece * kSplitThreads + tid, step = pieces * kSplitThreads;
    if (row == b * NKV && at == 0) keep_lens[b] = ctx < budget ? ctx : budget;
    if (ctx <= budget) {
      for (int i = at; i < budget; i += step) out[i] = i < ctx ? i : -1;
    } else {
      for (int i = at; i < sink; i += step) out[i] = i;
      for (int i = at; i < recent; i += step) out[budget - recent + i] = ctx - recent + i;
    }
  }
  if (ctx <= budget || n == 0) return;
  const float* s = scores + static_cast<size_t>(row) * cap + sink;
  const int count = ctx - recent - sink;  // candidates, more than n
  const int used = (count + kPiece - 1) / kPiece;
  if (piece >= used) return;
  uint32_t key[kSplitE];
  const int first = (piece * kWaves + wv) * (kSplitE * kWave) + lane;
  load_keys<kSplitE>(s, first, count, key);
  const SplitRow w(ws, row, pieces);

  uint32_t prefix = 0, mask = 0;
  int need = n;
#pragma unroll
  for (int p = 0; p + 1 < PASS; ++p) {
    prefix |= static_cast<uint32_t>(uniform(w.found[2 * p])) << digit_shift(p);
    mask |= static_cast<uint32_t>(digit_bins(p) - 1) << digit_shift(p);
    need -= uniform(w.found[2 * p + 1]);
  }
  int at = 0, same = 0;  // in the pieces before this one: kept, and equal to the key
  bool all_equal = false;
  if constexpr (PASS > 0) {
    constexpr int kPer = kBins / kSplitThreads;
    constexpr int p = PASS - 1;
    const int bins = digit_bins(p), per = bins / kSplitThreads;
    const int* counts = w.hist + static_cast<size_t>(p) * pieces * kBins;
    int mine[kPer] = {}, before[kPer] = {}, here[kPer] = {};
    const int low = bins - per * (tid + 1);  // this thread's bins, ascending
    for (int c = 0; c < used; ++c) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (j < per) {
          const int v = counts[c * kBins + low + per - 1 - j];
          mine[j] += v;
          before[j] += c < piece ? v : 0;
          here[j] = c == piece ? v : here[j];
        }
      }
    }
    find_digit<kSplitThreads>(mine, bins, need, part, found);
    const int digit = found[0];
    prefix |= static_cast<uint32_t>(digit) << digit_shift(p);
    mask |= static_cast<uint32_t>(bins - 1) << digit_shift(p);
    need -= found[1];
    // sums over the bins above the digit: of this piece, for pass 3; there, of those before
    int up = 0, eq = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int bin = low + per - 1 - j;
      if (j < per) {
        up += bin > digit ? (PASS == 3 ? before[j] : here[j]) : 0;
        eq += bin == digit ? before[j] : 0;
      }
    }
    up = wave_inclusive_scan(up, lane);
    eq = wave_inclusive_scan(eq, lane);
    if (lane == kWave - 1) {
      kept_tot[wv] = up;
      equal_tot[wv] = eq;
    }
    __syncthreads();
    int up_all, eq_all;
    before_wave<kWaves>(kept_tot, wv, lane, up_all);
    before_wave<kWaves>(equal_tot, wv, lane, eq_all);
    if constexpr (PASS < 3) {
      if (tid == 0) {
        w.above[p * pieces + piece] = up_all;
        if (piece == 0) {
          w.found[2 * p] = digit;
          w.found[2 * p + 1] = found[1];
        }
      }
    } else {
      all_equal = prefix != 0 && need == found[2];
      at = up_all;
      same = eq_all;
      for (int c = 0; c < piece; ++c) at += w.above[c] + w.above[pieces + c];
      if (all_equal) {  // (then they count as kept)
        at += same;
        same = 0;
      }
    }
  }
  if constexpr (PASS == 3) {
    write_kept<kSplitThreads, kSplitE>(key, first, count, prefix, need, all_equal, sink, out,
                                       kept_tot, equal_tot, at, same);
  } else {
    const int shift = digit_shift(PASS), bins = digit_bins(PASS);
    for (int i = tid; i < bins * kCopies; i += kSplitThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kSplitE; ++e) {
      if (first + e * kWave < count && (key[e] & mask) == prefix)
        atomicAdd(&hist[(key[e] >> shift) & (bins - 1)][lane % kCopies], 1);
    }
    __syncthreads();
    int* counts = w.hist + (static_cast<size_t>(PASS) * pieces + piece) * kBins;
    for (int i = tid; i < bins; i += kSplitThreads) {
      int sum = 0;
#pragma unroll
      for (int k = 0; k < kCopies; ++k) sum += hist[i][k];
      counts[i] = sum;
    }
  }
}

// ---- compaction ----------------------------------------------------------------
//
// Row start + i of a (sequence, kv head) takes row keep[i], K and V (and the score),
// ascending keep, keep[i] >= start + i where the pages are the same ones.
//
// One workgroup moves some dims of a head's rows: of K, or of V, whose 32-token blocks
// are transposed.  It reads a step of 512 rows into registers, waits until all of it is
// read, and writes: a later step's sources lie behind every row written so far, so the
// move may be in place, and the next step's rows, and the places of the two after it,
// are asked for before a step is written.  A step waits for its rows alone, not for the
// stores behind them (16 x 8 heads, half of 4,096 tokens, from memory: 68 us, with stores
// in the wait 79).
//
// A list that writes none of its own pages is moved in pieces by workgroups of their own,
// as many as make kFull segments (8 heads, 8,192 of 32,768 tokens: 34 us, in one piece 52;
// 4 x 8 heads, 4,096 of up to 16,384: 42 and 52, in four pieces 45).
//
// What bounds it: the kept rows read and written once; a V block is read in lines of
// 32 tokens of a dim, whichever of them stay.  64 dims of K and 16 of V per workgroup,
// since smaller pieces read lines of K more than once (16 x 8 heads, half of 4,096 tokens:
// 68 against 75 us with half of both); half of both where fewer than kFull segments leave
// CUs idle (in place; 8 heads, 7,000 of 8,192 tokens: 39 against 47 us).

constexpr int kMoveThreads = 512;
constexpr int kStep = 512;  // rows of a step
constexpr int kFull = 64;   // segments that fill the card
static_assert(kStep == kMoveThreads, "a thread looks one row up");

constexpr uint32_t kNoRow = 0xffffffffu;

struct CompactArgs {
  uint16_t* k_pool;
  uint16_t* v_pool;
  const int32_t* table;      // [B, max_pages]
  const int32_t* dst_table;  // [B, dst_pages]
  const int32_t* keep;       // [B, keep_heads, n]
  const int32_t* keep_lens;  // [B]
  const int32_t* start;      // [B], or null: 0
  const float* scores;       // [B, NKV, cap], or null
  float* scores_out;
  int NKV, D, keep_heads, n, cap, max_pages, dst_pages, pt_shift, num_slots;
  int chunks, chunk_steps;  // pieces of a list that goes to other pages, and their steps
};

// Page of a position within a table of so many (clamped: what lies outside is not used).
__device__ __forceinline__ int page_of(long long pos, int pages, const CompactArgs& a) {
  const long long page = pos >> a.pt_shift;
  return page < 0 ? 0 : (page < pages ? static_cast<int>(page) : pages - 1);
}

// Row of the pool (slot, kv head, token) of a position, in units of D elements.
__device__ __forceinline__ uint32_t row_of(int slot, long long pos, int pages, int kvh,
                                           const CompactArgs& a) {
  const bool ok = pos >= 0 && pos >> a.pt_shift < pages &&
                  static_cast<unsigned>(slot) < static_cast<unsigned>(a.num_slots);
  const uint32_t row = ((static_cast<uint32_t>(slot) * a.NKV + kvh) << a.pt_shift) +
                       (static_cast<uint32_t>(pos) & ((1u << a.pt_shift) - 1));
  return ok ? row : kNoRow;
}

// Where row i of the list is read and written; kNoRow: nothing to move.
__device__ __forceinline__ void look_up(const CompactArgs& a, const int32_t* keep, int n, int start,
                                        int b, int kvh, int i, uint32_t& src, uint32_t& dst) {
  const int32_t* trow = a.table + static_cast<size_t>(b) * a.max_pages;
  const int32_t* drow = a.dst_table + static_cast<size_t>(b) * a.dst_pages;
  const long long to = start + static_cast<long long>(i);
  const int d_slot = drow[page_of(to, a.dst_pages, a)];
  const int from = keep[i < n ? i : n - 1];
  const int s_slot = trow[page_of(from, a.max_pages, a)];
  const uint32_t s = row_of(s_slot, from, a.max_pages, kvh, a);
  const uint32_t d = row_of(d_slot, to, a.dst_pages, kvh, a);
  src = i >= n || d == kNoRow || d == s ? kNoRow : s;
  dst = d;
}

// The values are loaded here, not later.
template <typename T, int N>
__device__ __forceinline__ void pin(T (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+v"(v[j]));
}

// Every load of this wavefront has landed, and nothing moves across.
__device__ __forceinline__ void all_read() {
  wait_vmem_all();
  __syncthreads();
}

// Element of V(row, d) = block row / VB of [D, VB], VB = 1 << vb = min(page, 32).
__device__ __forceinline__ size_t v_element(uint32_t row, int d, int vb, int D) {
  return ((static_cast<size_t>(row >> vb) * D + d) << vb) + (row & ((1u << vb) - 1));
}

// One workgroup: the scores of one (sequence, kv head), and zeros behind them.
//
// In one array a round of kRound rows may only write what no later round reads.  Since the
// list ascends, keep[i] - i never falls: a first part of the rows, which may be empty, moves
// back (keep[i] < start + i) and goes from its end, the others from their front.  Where one
// round holds the list it is read as a whole.
template <int THREADS>
__device__ __forceinline__ void move_scores(const CompactArgs& a, const int32_t* keep, int b,
                                            int kvh, int n, int start) {
  const int tid = static_cast<int>(threadIdx.x);
  const size_t row = (static_cast<size_t>(b) * a.NKV + kvh) * a.cap;
  const float* s = a.scores + row;
  float* o = a.scores_out + row;
  const int first = start < a.cap ? start : a.cap;
  if (s != o)
    for (int i = tid; i < first; i += THREADS) o[i] = s[i];
  constexpr int kLoads = 8;
  constexpr int kRound = kLoads * THREADS;
  auto moves_back = [&](int i) { return keep[i] < start + static_cast<long long>(i); };
  int back = 0;  // rows that move back
  if (s == o && n > kRound && moves_back(0)) {
    int not_back = n;
    while (back < not_back) {
      const int i = back + (not_back - back) / 2;
      if (moves_back(i)) back = i + 1;
      else not_back = i;
    }
    back = uniform(back);
  }
  auto round = [&](int i0, int end) {
    int from[kLoads];
    float v[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = i0 + j * THREADS + tid;
      from[j] = i < end ? keep[i] : -1;
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) v[j] = from[j] >= 0 && from[j] < a.cap ? s[from[j]] : 0.f;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) asm volatile("" : "+v"(v[j]));
    all_read();
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = i0 + j * THREADS + tid;
      if (i < end && start + static_cast<long long>(i) < a.cap) o[start + i] = v[j];
    }
  };
  for (int i1 = back; i1 > 0; i1 -= kRound) round(i1 > kRound ? i1 - kRound : 0, i1);
  for (int i0 = back; i0 < n; i0 += kRound) round(i0, n);
  for (long long i = static_cast<long long>(first) + n + tid; i < a.cap; i += THREADS)
    o[i] = 0.f;
}

template <int kKDims, int kVDims>
__global__ __launch_bounds__(kMoveThreads) void compact_kernel(CompactArgs a) {
  // Places of the step being written, the one being read, and the one looked up.
  // As offsets in bytes of a row's first element: of K, or of V.
  __shared__ uint64_t src[4][kStep], dst[4][kStep];
  __shared__ bool ok[kStep];
  __shared__ int bad[4];  // the step has rows outside the tables or the pool
  const int tid = static_cast<int>(threadIdx.x);
  const int kvh = static_cast<int>(blockIdx.y);
  const int b = static_cast<int>(blockIdx.z);
  const int k_parts = (a.D + kKDims - 1) / kKDims, v_parts = a.D / kVDims;
  const int chunk = static_cast<int>(blockIdx.x) / (k_parts + v_parts);
  const int part = static_cast<int>(blockIdx.x) - chunk * (k_parts + v_parts);
  const int32_t* keep = a.keep + (static_cast<size_t>(b) * a.keep_heads +
                                  (a.keep_heads == 1 ? 0 : kvh)) * a.n;
  int n = uniform(a.keep_lens[b]);
  n = n < 0 ? 0 : (n > a.n ? a.n : n);
  int start = a.start != nullptr ? uniform(a.start[b]) : 0;
  start = start < 0 ? 0 : start;
  if (chunk == a.chunks) {
    move_scores<kMoveThreads>(a, keep, b, kvh, n, start);
    return;
  }
  const int32_t* trow = a.table + static_cast<size_t>(b) * a.max_pages;
  const int32_t* drow = a.dst_table + static_cast<size_t>(b) * a.dst_pages;
  int s = 0, steps = (n + kStep - 1) / kStep;  // the steps s .. steps are this workgroup's
  if (a.chunks > 1) {
    // a list that writes none of its own pages is moved in pieces, at the same time
    bool own = false;
    const long long to = start + static_cast<long long>(n) - 1;
    for (long long p = (start >> a.pt_shift) + tid; p <= to >> a.pt_shift; p += kMoveThreads)
      own |= p < a.max_pages && p < a.dst_pages && trow[p] == drow[p];
    if (__syncthreads_or(own) == 0) {
      s = chunk * a.chunk_steps;
      steps = min(steps, s + a.chunk_steps);
      n = min(n, steps * kStep);
    } else if (chunk != 0) {
      return;
    }
  }
  if (s >= steps) return;

  constexpr int kKPass = kMoveThreads / (kKDims / 8), kVPass = kMoveThreads / kVDims;
  constexpr int kKLoads = kStep / kKPass, kVLoads = kStep / kVPass;
  int kc = part * kKDims + 8 * (tid % (kKDims / 8));
  kc = kc < a.D ? kc : a.D - 8;  // (moved twice, the same values)
  const int vb = a.pt_shift < 5 ? a.pt_shift : 5;
  const int vd = (part - k_parts) * kVDims + tid / kVPass;
  // Row tid of step s (past the last one: that one again, the same values).
  auto index_of = [&](int s) {
    const int i = s * kStep + tid;
    return i < n ? i : n - 1;
  };
  struct Slots {
    int from, src, dst;
  };
  auto slots_of = [&](int s, int from) {
    const long long to = start + static_cast<long long>(index_of(s));
    return Slots{from, trow[page_of(from, a.max_pages, a)], drow[page_of(to, a.dst_pages, a)]};
  };
  const bool keys = part < k_parts;
  auto set_places = [&](int s, const Slots& x) {
    const long long at = start + static_cast<long long>(index_of(s));
    const uint32_t from = row_of(x.src, x.from, a.max_pages, kvh, a);
    const uint32_t to = row_of(x.dst, at, a.dst_pages, kvh, a);
    const int shift = keys ? 0 : vb;
    src[s & 3][tid] = v_element(from, 0, shift, a.D) * 2;
    dst[s & 3][tid] = v_element(to, 0, shift, a.D) * 2;
    const bool in_pool = from != kNoRow && to != kNoRow;
    ok[tid] = in_pool;
    if (!in_pool) bad[s & 3] = 1;
    return from != to;
  };
  // (the address is one addition: with the products here a step was bound by them)
  char* const k_base = reinterpret_cast<char*>(a.k_pool + kc);
  char* const v_base = reinterpret_cast<char*>(a.v_pool + (static_cast<size_t>(vd) << vb));
  auto read_k = [&](uint64_t from, u32x4& v) {
    v = *reinterpret_cast<const u32x4*>(k_base + from);
  };
  auto write_k = [&](uint64_t to, const u32x4& v) { *reinterpret_cast<u32x4*>(k_base + to) = v; };
  auto read_v = [&](uint64_t from, uint32_t& v) {
    v = *reinterpret_cast<const uint16_t*>(v_base + from);
  };
  auto write_v = [&](uint64_t to, uint32_t v) {
    *reinterpret_cast<uint16_t*>(v_base + to) = static_cast<uint16_t>(v);
  };
  // A thread's rows of a step are first, first + stride ...
  auto run = [&](auto& even, auto& odd, int first, int stride, auto read, auto write) {
    constexpr int kLoads = sizeof(even) / sizeof(even[0]);
    if (tid < 4) bad[tid] = 0;
    __syncthreads();
    // steps whose rows stay where they are (of a sequence within its budget: all)
    while (__syncthreads_or(set_places(s, slots_of(s, keep[index_of(s)]))) == 0)
      if (++s == steps) return;
    if (bad[s & 3] == 0) {
      auto load = [&](int t, auto& v) {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) read(src[t & 3][first + j * stride], v[j]);
      };
      Slots ahead = slots_of(s + 1, keep[index_of(s + 1)]);
      int from = keep[index_of(s + 2)];
      load(s, even);
      pin(even);
      // (no load or store here depends on a branch, and a step ends where its rows are
      // waited for: that wait then does not include the stores behind them)
      auto step = [&](auto& cur, auto& next) {
        set_places(s + 1, ahead);
        lds_barrier();  // every wavefront has read step s
        const bool go_on = bad[(s + 1) & 3] == 0;
        if (go_on) {
          ahead = slots_of(s + 2, from);
          from = keep[index_of(s + 3)];
          load(s + 1, next);
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) write(dst[s & 3][first + j * stride], cur[j]);
        pin(next);
        return ++s < steps && go_on;
      };
      while (step(even, odd) && step(odd, even)) {
      }
    }
    for (; s < steps; ++s) {  // (tables that name places outside the pool)
      __syncthreads();
      set_places(s, slots_of(s, keep[index_of(s)]));
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int at = first + j * stride;
        if (ok[at]) read(src[s & 3][at], even[j]);
      }
      pin(even);
      all_read();
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int at = first + j * stride;
        if (ok[at]) write(dst[s & 3][at], even[j]);
      }
    }
  };
  if (part < k_parts) {
    u32x4 even[kKLoads], odd[kKLoads];
    run(even, odd, tid / (kKDims / 8), kKPass, read_k, write_k);
  } else {
    uint32_t even[kVLoads], odd[kVLoads];
    run(even, odd, tid % kVPass, kVPass, read_v, write_v);
  }
}

// Few rows (the accepted branch of a tree of drafts): one workgroup per (sequence, kv
// head) moves all of them, every row of 128 dims read before the first is written.
constexpr int kFewRows = 64;
constexpr int kFewDims = 128;

__global__ __launch_bounds__(kMoveThreads) void compact_few_kernel(CompactArgs a) {
  __shared__ uint32_t src[kFewRows], dst[kFewRows];
  const int tid = static_cast<int>(threadIdx.x);
  const int kvh = static_cast<int>(blockIdx.y);
  const int b = static_cast<int>(blockIdx.z);
  const int32_t* keep = a.keep + (static_cast<size_t>(b) * a.keep_heads +
                                  (a.keep_heads == 1 ? 0 : kvh)) * a.n;
  int n = uniform(a.keep_lens[b]);
  n = n < 0 ? 0 : (n > a.n ? a.n : n);
  int start = a.start != nullptr ? uniform(a.start[b]) : 0;
  start = start < 0 ? 0 : start;
  if (blockIdx.x == 1) {
    move_scores<kMoveThreads>(a, keep, b, kvh, n, start);
    return;
  }
  if (n == 0) return;
  if (tid < n) look_up(a, keep, n, start, b, kvh, tid, src[tid], dst[tid]);
  __syncthreads();
  const int vb = a.pt_shift < 5 ? a.pt_shift : 5;
  for (int d0 = 0; d0 < a.D; d0 += kFewDims) {
    const int dims = a.D - d0 < kFewDims ? a.D - d0 : kFewDims;
    constexpr int kLoads = kFewRows * kFewDims / 8 / kMoveThreads;  // K, 16 bytes each
    constexpr int kColumns = kFewRows * kFewDims / kMoveThreads;    // V, elements
    const int chunk = tid % (kFewDims / 8), r0 = tid / (kFewDims / 8);
    u32x4 k[kLoads];
    uint32_t v[kColumns];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = r0 + j * (kMoveThreads / (kFewDims / 8));
      if (i < n && 8 * chunk < dims && src[i] != kNoRow)
        k[j] = *reinterpret_cast<const u32x4*>(a.k_pool + static_cast<size_t>(src[i]) * a.D + d0 +
                                               8 * chunk);
    }
#pragma unroll
    for (int j = 0; j < kColumns; ++j) {  // 16 rows side by side, 32 dims, rows slowest
      const int i = (tid & 15) + 16 * (j / (kFewDims / 32));
      const int d = tid / 16 + 32 * (j % (kFewDims / 32));
      if (i < n && d < dims && src[i] != kNoRow)
        v[j] = a.v_pool[v_element(src[i], d0 + d, vb, a.D)];
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) asm volatile("" : "+v"(k[j]));
#pragma unroll
    for (int j = 0; j < kColumns; ++j) asm volatile("" : "+v"(v[j]));
    all_read();
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = r0 + j * (kMoveThreads / (kFewDims / 8));
      if (i < n && 8 * chunk < dims && src[i] != kNoRow)
        *reinterpret_cast<u32x4*>(a.k_pool + static_cast<size_t>(dst[i]) * a.D + d0 + 8 * chunk) =
            k[j];
    }
#pragma unroll
    for (int j = 0; j < kColumns; ++j) {
      const int i = (tid & 15) + 16 * (j / (kFewDims / 32));
      const int d = tid / 16 + 32 * (j % (kFewDims / 32));
      if (i < n && d < dims && src[i] != kNoRow)
        a.v_pool[v_element(dst[i], d0 + d, vb, a.D)] = static_cast<uint16_t>(v[j]);
    }
  }
}

}  // namespace
}  // namespace voom

using namespace voom;

namespace {

// Pieces of a row in a call, 0: one workgroup takes the row.
int split_pieces(long long rows, int score_tokens) {
  const int pieces = (score_tokens + kPiece - 1) / kPiece;
  return score_tokens > kRowMost && pieces <= kMostPieces && rows <= kFewSplit ? pieces : 0;
}

bool select_shape_ok(int batch, int num_kv_heads, int score_tokens) {
  return batch > 0 && num_kv_heads > 0 && score_tokens > 0 && score_tokens < (1 << 30) &&
         static_cast<long long>(batch) * num_kv_heads < (1LL << 30);
}

}  // namespace

extern "C" size_t voom_evict_select_workspace_bytes(int batch, int num_kv_heads,
                                                    int score_tokens) {
  if (!select_shape_ok(batch, num_kv_heads, score_tokens)) return 0;
  const long long rows = static_cast<long long>(batch) * num_kv_heads;
  const int pieces = split_pieces(rows, score_tokens);
  return pieces == 0 ? 0 : rows * SplitRow::ints(pieces) * sizeof(int);
}

extern "C" int voom_evict_select(const float* scores, const int32_t* ctx_lens, int32_t* keep,
                                 int32_t* keep_lens, int batch, int num_kv_heads,
                                 int score_tokens, int budget, int sink, int recent,
                                 hipStream_t stream) {
  return voom_evict_select_split(scores, ctx_lens, keep, keep_lens, nullptr, 0, batch,
                                 num_kv_heads, score_tokens, budget, sink, recent, stream);
}

extern "C" int voom_evict_select_split(const float* scores, const int32_t* ctx_lens,
                                       int32_t* keep, int32_t* keep_lens, void* workspace,
                                       size_t ws_bytes, int batch, int num_kv_heads,
                                       int score_tokens, int budget, int sink, int recent,
                                       hipStream_t stream) {
  const char* who = "evict_select";
  VOOM_REQUIRE(scores && ctx_lens && keep && keep_lens, "%s: null pointer argument", who);
  VOOM_REQUIRE(select_shape_ok(batch, num_kv_heads, score_tokens),
               "%s: unsupported geometry (batch %d, %d kv heads, %d tokens)", who, batch,
               num_kv_heads, score_tokens);
  VOOM_REQUIRE(budget > 0 && sink >= 0 && recent >= 0 && sink <= budget && recent <= budget - sink,
               "%s: sink %d and recent %d must fit the budget %d", who, sink, recent, budget);
  const size_t need = voom_evict_select_workspace_bytes(batch, num_kv_heads, score_tokens);
  if (workspace != nullptr && need != 0) {
    VOOM_REQUIRE(ws_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "%s: workspace %zu bytes < required %zu (16-byte aligned)", who, ws_bytes, need);
    const int pieces = split_pieces(static_cast<long long>(batch) * num_kv_heads, score_tokens);
    const auto pass = [&](auto kernel) {
      hipLaunchKernelGGL(kernel,
                         dim3(static_cast<unsigned>(pieces),
                              static_cast<unsigned>(batch * num_kv_heads)),
                         dim3(kSplitThreads), 0, stream, scores, ctx_lens, keep, keep_lens,
                         static_cast<int*>(workspace), num_kv_heads, score_tokens, budget, sink,
                         recent, pieces);
    };
    pass(evict_split_kernel<0>);
    pass(evict_split_kernel<1>);
    pass(evict_split_kernel<2>);
    pass(evict_split_kernel<3>);
    return VOOM_LAUNCH_CHECK("evict_select: launch");
  }
  const auto launch = [&](auto kernel, int threads) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(batch * num_kv_heads)), dim3(threads), 0,
                       stream, scores, ctx_lens, keep, keep_lens, num_kv_heads, score_tokens,
                       budget, sink, recent);
  };
  if (score_tokens <= 8 * 256) launch(evict_select_kernel<256, 8, 1>, 256);
  else if (score_tokens <= 8 * 1024) launch(evict_select_kernel<1024, 8, 2>, 1024);
  else launch(evict_select_kernel<1024, 32, 8>, 1024);
  return VOOM_LAUNCH_CHECK("evict_select: launch");
}

extern "C" int voom_compact_kv(void* k_pool, void* v_pool, const int32_t* block_table,
                               const int32_t* dst_table, const int32_t* keep,
                               const int32_t* keep_lens, const int32_t* start,
                               const float* scores, float* scores_out, int batch,
                               int num_kv_heads, int head_dim, int page_tokens, int max_pages,
                               int dst_pages, int num_slots, int keep_heads, int keep_tokens,
                               int score_tokens, hipStream_t stream) {
  const char* who = "compact_kv";
  VOOM_REQUIRE(k_pool && v_pool && block_table && dst_table && keep && keep_lens,
               "%s: null pointer argument", who);
  VOOM_REQUIRE(batch > 0 && batch <= 65535 && num_kv_heads > 0 && num_kv_heads <= 65535 &&
                   max_pages > 0 && dst_pages > 0 && num_slots > 0 && keep_tokens > 0 &&
                   keep_tokens < (1 << 30),
               "%s: bad geometry (batch %d, %d kv heads, %d rows)", who, batch, num_kv_heads,
               keep_tokens);
  VOOM_REQUIRE(head_dim > 0 && head_dim % 32 == 0, "%s: head_dim %d not a multiple of 32", who,
               head_dim);
  VOOM_REQUIRE(is_pow2(page_tokens) && page_tokens <= 4096,
               "%s: page_tokens %d must be a power of two <= 4096", who, page_tokens);
  VOOM_REQUIRE(static_cast<long long>(num_slots) * num_kv_heads * page_tokens < (1LL << 32) - 1,
               "%s: more than 2^32 - 2 rows in the pool", who);
  VOOM_REQUIRE(keep_heads == 1 || keep_heads == num_kv_heads, "%s: %d lists for %d kv heads", who,
               keep_heads, num_kv_heads);
  VOOM_REQUIRE((scores == nullptr) == (scores_out == nullptr) &&
                   (scores == nullptr || score_tokens > 0),
               "%s: scores and scores_out go together", who);
  VOOM_REQUIRE(reinterpret_cast<uintptr_t>(k_pool) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v_pool) % 16 == 0,
               "%s: pools must be 16-byte aligned", who);
  CompactArgs a;
  a.k_pool = static_cast<uint16_t*>(k_pool);
  a.v_pool = static_cast<uint16_t*>(v_pool);
  a.table = block_table;
  a.dst_table = dst_table;
  a.keep = keep;
  a.keep_lens = keep_lens;
  a.start = start;
  a.scores = scores;
  a.scores_out = scores_out;
  a.NKV = num_kv_heads;
  a.D = head_dim;
  a.keep_heads = keep_heads;
  a.n = keep_tokens;
  a.cap = score_tokens;
  a.max_pages = max_pages;
  a.dst_pages = dst_pages;
  a.pt_shift = ilog2(page_tokens);
  a.num_slots = num_slots;
  const unsigned moves_scores = scores != nullptr ? 1 : 0;
  dim3 grid(1 + moves_scores, static_cast<unsigned>(num_kv_heads), static_cast<unsigned>(batch));
  if (keep_tokens <= kFewRows) {
    hipLaunchKernelGGL(compact_few_kernel, grid, dim3(kMoveThreads), 0, stream, a);
  } else {
    const long long segs = static_cast<long long>(batch) * num_kv_heads;
    const int steps = (keep_tokens + kStep - 1) / kStep;
    const int pieces = dst_table == block_table || segs >= kFull
                           ? 1 : static_cast<int>((kFull + segs - 1) / segs);
    a.chunk_steps = (steps + pieces - 1) / pieces;
    a.chunks = (steps + a.chunk_steps - 1) / a.chunk_steps;
    const auto launch = [&](auto kernel, int k_dims, int v_dims) {
      grid.x = ((head_dim + k_dims - 1) / k_dims + head_dim / v_dims) * a.chunks + moves_scores;
      hipLaunchKernelGGL(kernel, grid, dim3(kMoveThreads), 0, stream, a);
    };
    if (segs * a.chunks >= kFull) launch(compact_kernel<64, 16>, 64, 16);
    else launch(compact_kernel<32, 8>, 32, 8);
  }
  return VOOM_LAUNCH_CHECK("compact_kv: launch");
}
