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
// workgroup per (sequence, head).  Up to 65,536 candidates stay in registers, all loads
// in flight at once (a loop that loaded them for every pass: 43 us for 16 x 8 heads of
// up to 32,768 tokens, where this takes TIME_SELECT); of longer ones every pass loads
// 65,536 at a time.  A histogram has eight copies, by lane: scores share few leading bits,
// and atomics of one wavefront on one address take turns.

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kBins = 2048;
constexpr int kCopies = 8;

// Larger score, larger key; NaN 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 + 0 is 0
  const uint32_t k = (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
  return x != x ? 0u : k;
}

// E: candidates per thread and round.  Round c, wavefront w, element e, lane l hold
// candidate ((c * 16 + w) * E + e) * 64 + l.
template <int E>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(
    const float* __restrict__ scores, const int32_t* __restrict__ ctx_lens,
    int32_t* __restrict__ keep, int32_t* __restrict__ keep_lens, int NKV, int cap, int budget,
    int sink, int recent) {
  __shared__ __attribute__((aligned(16))) int hist[kBins][kCopies];
  __shared__ int part[kSelWaves];
  __shared__ int found[2];  // digit that holds the n-th largest, keys above it in this pass
  __shared__ int above_tot[kSelWaves], equal_tot[kSelWaves];
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
  for (int i = tid; i < sink; i += kSelThreads) out[i] = i;
  for (int i = tid; i < recent; i += kSelThreads) out[budget - recent + i] = ctx - recent + i;
  const int n = budget - sink - recent;
  if (n == 0) return;
  const float* s = scores + static_cast<size_t>(row) * cap + sink;
  const int count = ctx - recent - sink;  // candidates, more than n
  const int rounds = (count + kSelThreads * E - 1) / (kSelThreads * E);

  uint32_t key[E];
  const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<float*>(s), static_cast<short>(0), count * 4, 0x00020000);  // past it: 0
  auto load = [&](int c) {
    const int first = (c * kSelWaves + wv) * (E * kWave) + lane;
#pragma unroll
    for (int e = 0; e < E; ++e)
      key[e] = __builtin_amdgcn_raw_buffer_load_b32(from, first * 4, e * (kWave * 4), 0);
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = order_key(__builtin_bit_cast(float, key[e]));
  };
  // the candidates of this wavefront's element e, round c
  auto inside = [&](int c, int e) {
    return ((c * kSelWaves + wv) * E + e) * kWave + lane < count;
  };
  load(0);

  uint32_t prefix = 0, mask = 0;  // the bits of the n-th largest key found so far
  int need = n;                   // its rank among the keys with that prefix
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int bins = pass == 2 ? 1024 : 2048;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int i = tid; i < kBins * kCopies / 4; i += kSelThreads)
      *reinterpret_cast<u32x4*>(&hist[0][0] + 4 * i) = zero;
    __syncthreads();
    for (int c = 0; c < rounds; ++c) {
      if (rounds > 1 && (pass > 0 || c > 0)) load(c);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (inside(c, e) && (key[e] & mask) == prefix)
          atomicAdd(&hist[(key[e] >> shift) & (bins - 1)][lane % kCopies], 1);
      }
    }
    __syncthreads();
    // thread t owns bins t * per .. of the descending order
    const int per = bins / kSelThreads;
    int mine[2] = {0, 0};
    for (int j = 0; j < per; ++j) {
      const int* h = hist[bins - 1 - (tid * per + j)];
      const u32x4 lo = *reinterpret_cast<const u32x4*>(h), hi = *reinterpret_cast<const u32x4*>(h + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) mine[j] += static_cast<int>(lo[k] + hi[k]);
    }
    const int x = wave_inclusive_scan(mine[0] + mine[1], lane);
    if (lane == kWave - 1) part[wv] = x;
    __syncthreads();
    int before = x - (mine[0] + mine[1]);
    for (int k = 0; k < wv; ++k) before += part[k];
    for (int j = 0; j < per; ++j) {
      if (before < need && before + mine[j] >= need) {
        found[0] = bins - 1 - (tid * per + j);
        found[1] = before;
      }
      before += mine[j];
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found[0]) << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    need -= found[1];
  }

  // `prefix` is the n-th largest key; `need` of those equal to it stay.  Each
  // wavefront counts its run of the candidates and writes behind the runs before it.
  int at = 0, same = 0;  // kept above the key, and equal to it, before the run
  for (int c = 0; c < rounds; ++c) {
    if (rounds > 1) load(c);
    int above = 0, equal = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      above += __popcll(__builtin_amdgcn_ballot_w64(inside(c, e) && key[e] > prefix));
      equal += __popcll(__builtin_amdgcn_ballot_w64(inside(c, e) && key[e] == prefix));
    }
    // (keeps the compiler from holding two lane masks per element until below)
#pragma unroll
    for (int e = 0; e < E; ++e) asm volatile("" : "+v"(key[e]));
    __syncthreads();  // the totals of the round before are read
    if (lane == 0) {
      above_tot[wv] = above;
      equal_tot[wv] = equal;
    }
    __syncthreads();
    int up_all = 0, eq_all = 0;
    for (int k = 0; k < kSelWaves; ++k) {
      if (k == wv) {
        above = up_all;
        equal = eq_all;
      }
      up_all += above_tot[k];
      eq_all += equal_tot[k];
    }
    int up_at = at + above, eq_at = same + equal;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = inside(c, e);
      const uint64_t up = __builtin_amdgcn_ballot_w64(in && key[e] > prefix);
      const uint64_t eq = __builtin_amdgcn_ballot_w64(in && key[e] == prefix);
      const uint64_t low = (1ull << lane) - 1;
      const int eq_before = eq_at + __popcll(eq & low);
      if (in && (key[e] > prefix || (key[e] == prefix && eq_before < need))) {
        const int eq_kept = eq_before < need ? eq_before : need;
        out[sink + up_at + __popcll(up & low) + eq_kept] =
            sink + ((c * kSelWaves + wv) * E + e) * kWave + lane;
      }
      up_at += __popcll(up);
      eq_at += __popcll(eq);
    }
    at += up_all;
    same += eq_all;
  }
}

// ---- compaction ----------------------------------------------------------------
//
// Row start + i of a (sequence, kv head) takes row keep[i], K and V (and the score),
// ascending keep, keep[i] >= start + i where the pages are the same ones.
//
// One workgroup moves some dims of a head's rows: 32 dims (64 bytes) of K, or 16 dims
// of V, whose 32-token blocks are transposed.  It reads a step's rows into registers,
// waits until all of it is read, and writes: a later step's sources lie behind every
// row written so far, so the move may be in place.  The next step's places are looked
// up while its rows come.
//
// What bounds it: the kept rows read and written once; a V block is read in lines of
// 32 tokens of a dim, whichever of them stay.

constexpr int kMoveThreads = 512;
constexpr int kStep = 512;  // rows of a step
constexpr int kKDims = 32, kVDims = 16;
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
};

// Row of the pool (slot, kv head, token) of a position, in units of D elements.
__device__ __forceinline__ uint32_t row_of(const int32_t* table, int pages, int pos, int kvh,
                                           const CompactArgs& a) {
  if (pos < 0) return kNoRow;
  const int page = pos >> a.pt_shift;
  if (page >= pages) return kNoRow;
  const int slot = table[page];
  if (static_cast<unsigned>(slot) >= static_cast<unsigned>(a.num_slots)) return kNoRow;
  return ((static_cast<uint32_t>(slot) * a.NKV + kvh) << a.pt_shift) +
         (pos & ((1 << a.pt_shift) - 1));
}

// Every load of this wavefront has landed, and nothing moves across.
__device__ __forceinline__ void all_read() {
  wait_vmem_all();
  __syncthreads();
}

// Where position `from` is read and position `to` written; kNoRow: nothing to move.
__device__ __forceinline__ void places(const CompactArgs& a, const int32_t* trow,
                                       const int32_t* drow, int from, long long to, int kvh,
                                       uint32_t& src, uint32_t& dst) {
  const uint32_t s = row_of(trow, a.max_pages, from, kvh, a);
  const uint32_t d =
      to < (1LL << 30) ? row_of(drow, a.dst_pages, static_cast<int>(to), kvh, a) : kNoRow;
  src = d == kNoRow || d == s ? kNoRow : s;
  dst = d;
}

// Element of V(row, d) = block row / VB of [D, VB], VB = 1 << vb = min(page, 32).
__device__ __forceinline__ size_t v_element(uint32_t row, int d, int vb, int D) {
  return ((static_cast<size_t>(row >> vb) * D + d) << vb) + (row & ((1u << vb) - 1));
}

// One workgroup: the scores of one (sequence, kv head), and zeros behind them.
__device__ __forceinline__ void move_scores(const CompactArgs& a, const int32_t* keep, int b,
                                            int kvh, int n, int start) {
  const int tid = static_cast<int>(threadIdx.x);
  const size_t row = (static_cast<size_t>(b) * a.NKV + kvh) * a.cap;
  const float* s = a.scores + row;
  float* o = a.scores_out + row;
  const int first = start < a.cap ? start : a.cap;
  if (s != o)
    for (int i = tid; i < first; i += kMoveThreads) o[i] = s[i];
  constexpr int kLoads = 8;
  for (int i0 = 0; i0 < n; i0 += kLoads * kMoveThreads) {
    int from[kLoads];
    float v[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = i0 + j * kMoveThreads + tid;
      from[j] = i < n ? keep[i] : -1;
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) v[j] = from[j] >= 0 && from[j] < a.cap ? s[from[j]] : 0.f;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) asm volatile("" : "+v"(v[j]));
    all_read();
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int i = i0 + j * kMoveThreads + tid;
      if (i < n && start + static_cast<long long>(i) < a.cap) o[start + i] = v[j];
    }
  }
  for (long long i = static_cast<long long>(first) + n + tid; i < a.cap; i += kMoveThreads)
    o[i] = 0.f;
}

__global__ __launch_bounds__(kMoveThreads) void compact_kernel(CompactArgs a) {
  static_assert(kStep == kMoveThreads, "a thread looks one row up");
  // Places of three steps: while the next step's are looked up, a wavefront may still
  // store the rows of the step before.
  __shared__ uint32_t src[3][kStep], dst[3][kStep];
  const int tid = static_cast<int>(threadIdx.x);
  const int kvh = static_cast<int>(blockIdx.y);
  const int b = static_cast<int>(blockIdx.z);
  const int k_parts = a.D / kKDims, v_parts = a.D / kVDims;
  const int part = static_cast<int>(blockIdx.x);
  const int32_t* keep = a.keep + (static_cast<size_t>(b) * a.keep_heads +
                                  (a.keep_heads == 1 ? 0 : kvh)) * a.n;
  int n = uniform(a.keep_lens[b]);
  n = n < 0 ? 0 : (n > a.n ? a.n : n);
  int start = a.start != nullptr ? uniform(a.start[b]) : 0;
  start = start < 0 ? 0 : start;

  if (part == k_parts + v_parts) {
    move_scores(a, keep, b, kvh, n, start);
    return;
  }

  const int32_t* trow = a.table + static_cast<size_t>(b) * a.max_pages;
  const int32_t* drow = a.dst_table + static_cast<size_t>(b) * a.dst_pages;
  auto look_up = [&](int i0, int buf) {
    const int i = i0 + tid;
    if (i >= n) return;
    places(a, trow, drow, keep[i], start + static_cast<long long>(i), kvh, src[buf][tid],
           dst[buf][tid]);
  };
  look_up(0, 0);
  __syncthreads();
  int buf = 0, next = 1;
  for (int i0 = 0; i0 < n; i0 += kStep) {
    const int m = n - i0 < kStep ? n - i0 : kStep;
    if (part < k_parts) {
      constexpr int kChunks = kKDims / 8;
      constexpr int kPass = kMoveThreads / kChunks;
      constexpr int kLoads = kStep / kPass;
      const int c = part * kKDims + 8 * (tid % kChunks);
      const int r = tid / kChunks;
      u32x4 v[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const uint32_t from = r + j * kPass < m ? src[buf][r + j * kPass] : kNoRow;
        if (from != kNoRow)
          v[j] = *reinterpret_cast<const u32x4*>(a.k_pool + static_cast<size_t>(from) * a.D + c);
      }
      look_up(i0 + kStep, next);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) asm volatile("" : "+v"(v[j]));
      all_read();
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = r + j * kPass;
        if (i < m && src[buf][i] != kNoRow)
          *reinterpret_cast<u32x4*>(a.k_pool + static_cast<size_t>(dst[buf][i]) * a.D + c) = v[j];
      }
    } else {
      constexpr int kLoads = kStep / 32;
      const int vb = a.pt_shift < 5 ? a.pt_shift : 5;
      const int d = (part - k_parts) * kVDims + tid / 32;
      uint32_t v[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = (tid & 31) + 32 * j;
        const uint32_t from = i < m ? src[buf][i] : kNoRow;
        if (from != kNoRow) v[j] = a.v_pool[v_element(from, d, vb, a.D)];
      }
      look_up(i0 + kStep, next);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) asm volatile("" : "+v"(v[j]));
      all_read();
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = (tid & 31) + 32 * j;
        if (i < m && src[buf][i] != kNoRow)
          a.v_pool[v_element(dst[buf][i], d, vb, a.D)] = static_cast<uint16_t>(v[j]);
      }
    }
    buf = next;
    next = next == 2 ? 0 : next + 1;
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
    move_scores(a, keep, b, kvh, n, start);
    return;
  }
  if (tid < n)
    places(a, a.table + static_cast<size_t>(b) * a.max_pages,
           a.dst_table + static_cast<size_t>(b) * a.dst_pages, keep[tid],
           start + static_cast<long long>(tid), kvh, src[tid], dst[tid]);
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

extern "C" int voom_evict_select(const float* scores, const int32_t* ctx_lens, int32_t* keep,
                                 int32_t* keep_lens, int batch, int num_kv_heads,
                                 int score_tokens, int budget, int sink, int recent,
                                 hipStream_t stream) {
  const char* who = "evict_select";
  VOOM_REQUIRE(scores && ctx_lens && keep && keep_lens, "%s: null pointer argument", who);
  VOOM_REQUIRE(batch > 0 && num_kv_heads > 0 && score_tokens > 0 &&
                   score_tokens < (1 << 30) &&
                   static_cast<long long>(batch) * num_kv_heads < (1LL << 30),
               "%s: unsupported geometry (batch %d, %d kv heads, %d tokens)", who, batch,
               num_kv_heads, score_tokens);
  VOOM_REQUIRE(budget > 0 && sink >= 0 && recent >= 0 && sink <= budget && recent <= budget - sink,
               "%s: sink %d and recent %d must fit the budget %d", who, sink, recent, budget);
  const dim3 grid(static_cast<unsigned>(batch * num_kv_heads)), block(kSelThreads);
  if (score_tokens <= 8 * kSelThreads)
    hipLaunchKernelGGL(evict_select_kernel<8>, grid, block, 0, stream, scores, ctx_lens, keep,
                       keep_lens, num_kv_heads, score_tokens, budget, sink, recent);
  else if (score_tokens <= 32 * kSelThreads)
    hipLaunchKernelGGL(evict_select_kernel<32>, grid, block, 0, stream, scores, ctx_lens, keep,
                       keep_lens, num_kv_heads, score_tokens, budget, sink, recent);
  else
    hipLaunchKernelGGL(evict_select_kernel<64>, grid, block, 0, stream, scores, ctx_lens, keep,
                       keep_lens, num_kv_heads, score_tokens, budget, sink, recent);
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
    grid.x = head_dim / kKDims + head_dim / kVDims + moves_scores;
    hipLaunchKernelGGL(compact_kernel, grid, dim3(kMoveThreads), 0, stream, a);
  }
  return VOOM_LAUNCH_CHECK("compact_kv: launch");
}
