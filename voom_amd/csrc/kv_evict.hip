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
// What bounds it: the scores once, 4 bytes per token and head, and the latency of the
// four passes of one workgroup per (sequence, head).

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kBins = 2048;

// Larger score, larger key; NaN 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 + 0 is 0
  if (x != x) return 0u;
  return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(
    const float* __restrict__ scores, const int32_t* __restrict__ ctx_lens,
    int32_t* __restrict__ keep, int32_t* __restrict__ keep_lens, int NKV, int cap, int budget,
    int sink, int recent) {
  __shared__ int hist[kBins];
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
  const float* s = scores + static_cast<size_t>(row) * cap;
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
  const int lo = sink, hi = ctx - recent;  // more than n candidates

  uint32_t prefix = 0, mask = 0;  // the bits of the n-th largest key found so far
  int need = n;                   // its rank among the keys with that prefix
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const int bins = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kSelThreads) {
      const uint32_t k = order_key(s[i]);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
    }
    __syncthreads();
    // thread t owns bins t * per .. of the descending order
    const int per = bins / kSelThreads;
    int mine[2] = {0, 0};
    for (int j = 0; j < per; ++j) mine[j] = hist[bins - 1 - (tid * per + j)];
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
    __syncthreads();
  }

  // `prefix` is the n-th largest key; `need` of those equal to it stay.  Each
  // wavefront takes a run of the candidates, counts, and writes behind the runs
  // before its own.
  const int run = ((hi - lo + kSelWaves - 1) / kSelWaves + kWave - 1) & ~(kWave - 1);
  const int r0 = lo + wv * run;
  const int r1 = r0 + run < hi ? r0 + run : hi;
  int above = 0, equal = 0;
  for (int i = r0; i < r1; i += kWave) {
    const uint32_t k = i + lane < r1 ? order_key(s[i + lane]) : 0u;
    above += __popcll(__builtin_amdgcn_ballot_w64(i + lane < r1 && k > prefix));
    equal += __popcll(__builtin_amdgcn_ballot_w64(i + lane < r1 && k == prefix));
  }
  if (lane == 0) {
    above_tot[wv] = above;
    equal_tot[wv] = equal;
  }
  __syncthreads();
  int at = 0, same = 0;  // kept above the key, and equal to it, in the runs before
  for (int k = 0; k < wv; ++k) {
    at += above_tot[k];
    same += equal_tot[k];
  }
  for (int i = r0; i < r1; i += kWave) {
    const bool in = i + lane < r1;
    const uint32_t k = in ? order_key(s[i + lane]) : 0u;
    const uint64_t up = __builtin_amdgcn_ballot_w64(in && k > prefix);
    const uint64_t eq = __builtin_amdgcn_ballot_w64(in && k == prefix);
    const uint64_t low = (1ull << lane) - 1;
    const int eq_before = same + __popcll(eq & low);
    const bool take = in && (k > prefix || (k == prefix && eq_before < need));
    if (take) {
      const int eq_kept = eq_before < need ? eq_before : need;
      out[sink + at + __popcll(up & low) + eq_kept] = i + lane;
    }
    at += __popcll(up);
    same += __popcll(eq);
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
// row written so far, so the move may be in place.
//
// What bounds it: the kept rows read and written once; a V block is read in lines of
// 32 tokens of a dim, whichever of them stay.

constexpr int kMoveThreads = 512;
constexpr int kStep = 1024;  // rows of a step
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

__global__ __launch_bounds__(kMoveThreads) void compact_kernel(CompactArgs a) {
  __shared__ uint32_t src[kStep], dst[kStep];
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

  if (part == k_parts + v_parts) {  // the scores
    const size_t row = (static_cast<size_t>(b) * a.NKV + kvh) * a.cap;
    const float* s = a.scores + row;
    float* o = a.scores_out + row;
    const int first = start < a.cap ? start : a.cap;
    if (s != o)
      for (int i = tid; i < first; i += kMoveThreads) o[i] = s[i];
    for (int i0 = 0; i0 < n; i0 += kMoveThreads) {
      float v = 0.f;
      const int i = i0 + tid;
      if (i < n) {
        const int from = keep[i];
        if (from >= 0 && from < a.cap) v = s[from];
      }
      asm volatile("" : "+v"(v));
      all_read();
      if (i < n && start + static_cast<long long>(i) < a.cap) o[start + i] = v;
    }
    for (long long i = static_cast<long long>(first) + n + tid; i < a.cap; i += kMoveThreads)
      o[i] = 0.f;
    return;
  }

  const int32_t* trow = a.table + static_cast<size_t>(b) * a.max_pages;
  const int32_t* drow = a.dst_table + static_cast<size_t>(b) * a.dst_pages;
  for (int i0 = 0; i0 < n; i0 += kStep) {
    const int m = n - i0 < kStep ? n - i0 : kStep;
    for (int i = tid; i < m; i += kMoveThreads) {
      const long long to = static_cast<long long>(start) + i0 + i;
      uint32_t from = row_of(trow, a.max_pages, keep[i0 + i], kvh, a);
      const uint32_t at =
          to < (1LL << 30) ? row_of(drow, a.dst_pages, static_cast<int>(to), kvh, a) : kNoRow;
      if (at == kNoRow || at == from) from = kNoRow;  // nothing to move
      src[i] = from;
      dst[i] = at;
    }
    __syncthreads();
    if (part < k_parts) {
      constexpr int kChunks = kKDims / 8;
      constexpr int kPass = kMoveThreads / kChunks;
      constexpr int kLoads = kStep / kPass;
      const int c = part * kKDims + 8 * (tid % kChunks);
      const int r = tid / kChunks;
      u32x4 v[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = r + j * kPass;
        const uint32_t from = i < m ? src[i] : kNoRow;
        if (from != kNoRow)
          v[j] = *reinterpret_cast<const u32x4*>(a.k_pool + static_cast<size_t>(from) * a.D + c);
      }
#pragma unroll
      for (int j = 0; j < kLoads; ++j) asm volatile("" : "+v"(v[j]));
      all_read();
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = r + j * kPass;
        if (i < m && src[i] != kNoRow)
          *reinterpret_cast<u32x4*>(a.k_pool + static_cast<size_t>(dst[i]) * a.D + c) = v[j];
      }
    } else {
      // V(row, d) = block row / VB of [D, VB], VB = min(page, 32)
      constexpr int kLoads = kStep / 32;
      const int vb = a.pt_shift < 5 ? a.pt_shift : 5;
      const int d = (part - k_parts) * kVDims + tid / 32;
      auto at = [&](uint32_t row) {
        return a.v_pool + (((static_cast<size_t>(row >> vb) * a.D) + d) << vb) +
               (row & ((1u << vb) - 1));
      };
      uint32_t v[kLoads];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = (tid & 31) + 32 * j;
        const uint32_t from = i < m ? src[i] : kNoRow;
        if (from != kNoRow) v[j] = *at(from);
      }
#pragma unroll
      for (int j = 0; j < kLoads; ++j) asm volatile("" : "+v"(v[j]));
      all_read();
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const int i = (tid & 31) + 32 * j;
        if (i < m && src[i] != kNoRow) *at(dst[i]) = static_cast<uint16_t>(v[j]);
      }
    }
    __syncthreads();  // src and dst are written again
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
  hipLaunchKernelGGL(evict_select_kernel, dim3(static_cast<unsigned>(batch * num_kv_heads)),
                     dim3(kSelThreads), 0, stream, scores, ctx_lens, keep, keep_lens, num_kv_heads,
                     score_tokens, budget, sink, recent);
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
  const unsigned parts = head_dim / kKDims + head_dim / kVDims + (scores != nullptr ? 1 : 0);
  hipLaunchKernelGGL(compact_kernel,
                     dim3(parts, static_cast<unsigned>(num_kv_heads), static_cast<unsigned>(batch)),
                     dim3(kMoveThreads), 0, stream, a);
  return VOOM_LAUNCH_CHECK("compact_kv: launch");
}
