// Beam search over the paged cache for gfx950: the best continuations of a request's beams
// (voom_beam_select), and the cached tokens of beams that go on from another one
// (voom_fork_kv).
//
// Selection.  Beam j of K with score s_j (a sum of log-probabilities) and logits x_j over V
// tokens has the continuations
//   c(j, v) = s_j + x_j[v] - log sum_u exp x_j[u],
// one that has ended a single one, its end token at c = s_j.  The K largest of all K V stay,
// equal ones the lowest (j, v) first; one that is NaN, or of a beam whose score or sum is
// not finite, counts as -inf.  They differ by their row: the best continuation of a beam
// stays in the beam's row, the others, best first, take the rows of beams that nothing
// goes on from, lowest first.  So no row that is read for a copy is written.
//
// What bounds it: the logits read once; for one request the two launches and what each waits
// for.  beam_pieces_kernel takes a piece of a beam's logits, EACH of a lane: in registers,
// their maximum, their sum of exponentials and their K largest.  A wavefront's lanes are put
// into K groups or some more: the least of the groups' maxima has K logits at or above it, so
// nothing below the largest such bound of the four wavefronts is among the K largest of the
// piece, and the few logits that are not below it (about K log K) are listed in LDS and
// ranked by counting.  beam_merge_kernel, a workgroup per request, does the same with all
// pieces' lists, in 64 bits, where values of different beams meet.  16 requests of 8 beams over
// 128,256 fp32 logits: 14.8 us and 10.9 (medians of a trace), 26-28 a call; 33 with bounds from
// single lanes.
#include "common.h"

#include <cmath>

namespace voom {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxBeams = 32;
constexpr int kList = 1024;                // logits listed at most
constexpr int kMergeThreads = 512;

struct BeamArgs {
  const void* logits;       // [B, K, V]
  const float* scores;      // [B, K]
  const int64_t* last;      // [B, K], or null: none has ended
  int64_t end_token;
  const int32_t* shared;    // [B, K, K], or null
  const int32_t* ctx;       // [B]
  uint64_t* keys;           // [B * K, pieces, K]
  float2* sums;             // [B * K, pieces]: maximum, sum of exponentials less it
  float* scores_out;        // [B, K]
  int64_t* tokens;
  int32_t* parents;
  int32_t* first;           // [B, K]
  int32_t* shared_out;      // [B, K, K]
  int B, K, V, pieces, groups;
};

// Ordered as the floats are; 0 is no value.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// A logit and its token: larger logits first, of equal ones lower tokens.  +0 and -0 are
// equal.
__device__ __forceinline__ uint64_t key_of(uint32_t k, int token) {
  return static_cast<uint64_t>(k) << 32 | (0xffffffffu - static_cast<uint32_t>(token));
}
__device__ __forceinline__ int token_of(uint64_t key) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
}

__device__ __forceinline__ bool ended(const BeamArgs& a, int row) {
  return a.last != nullptr && a.last[row] == a.end_token;
}

// A value that K lanes or more hold at least: the least of the maxima of `groups` groups of
// lanes, a power of two >= K.
template <class T>
__device__ __forceinline__ T lane_bound(T v, int groups) {
  for (int k = 1; k < kWave / groups; k <<= 1) {
    const T o = __shfl_xor(v, k);
    v = o > v ? o : v;
  }
  for (int k = kWave / groups; k < kWave; k <<= 1) {
    const T o = __shfl_xor(v, k);
    v = o < v ? o : v;
  }
  return v;
}

template <class T>
__device__ __forceinline__ T wave_best(T v) {
#pragma unroll
  for (int k = 1; k < kWave; k <<= 1) {
    const T o = __shfl_xor(v, k);
    v = o > v ? o : v;
  }
  return v;
}

__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(uint16_t x) { return bf2f(x); }

// T: float, or uint16_t for bf16.
template <class T, int EACH>
__global__ __launch_bounds__(kThreads) void beam_pieces_kernel(BeamArgs a) {
  constexpr int kPer = 16 / sizeof(T);  // logits of 16 bytes
  constexpr int kEach = EACH;
  constexpr int kPiece = kThreads * kEach;
  struct Chunk {
    T x[kPer];
  };
  __shared__ uint64_t list[kList];
  __shared__ float bounds[kWaves];
  __shared__ float2 part[kWaves];
  __shared__ uint64_t winner[2][kWaves];
  __shared__ int listed;
  const int piece = static_cast<int>(blockIdx.x);
  const int row = static_cast<int>(blockIdx.y) * a.K + static_cast<int>(blockIdx.z);
  if (ended(a, row)) return;  // its one continuation needs no logits
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = uniform(threadIdx.x / kWave);
  if (threadIdx.x == 0) listed = 0;

  // A lane's logits go by their tokens, not by the row's alignment: rows of equal logits then
  // have equal sums to the last bit, and equal continuations stay equal.
  const T* const logits = static_cast<const T*>(a.logits) + static_cast<size_t>(row) * a.V;
  float x[kEach];
  int at[kEach / kPer];  // tokens of this lane's 16-byte pieces
#pragma unroll
  for (int i = 0; i < kEach / kPer; ++i) {
    at[i] = piece * kPiece + (i * kThreads + static_cast<int>(threadIdx.x)) * kPer;
    if (at[i] + kPer <= a.V) {
      Chunk v;  // (aligned as a logit is)
      __builtin_memcpy(&v, logits + at[i], sizeof(v));
#pragma unroll
      for (int e = 0; e < kPer; ++e) x[i * kPer + e] = value_of(v.x[e]);
    } else {
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        x[i * kPer + e] = at[i] + e < a.V ? value_of(logits[at[i] + e]) : -INFINITY;
    }
  }
  auto token = [&](int i) { return at[i / kPer] + i % kPer; };
  auto inside = [&](int i) { return token(i) < a.V; };

  // maximum and sum of this lane, then of the piece (a NaN makes the sum one, and then no
  // list of the beam is used)
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) m = fmaxf(m, x[i]);
  const float ref = m > -INFINITY ? m : 0.f;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) s += fast_exp2((x[i] - ref) * 1.4426950408889634f);
  const float top = wave_max_uniform(m);
  // (a lane of no logits or -inf alone has the sum 0, and no maximum that it could be scaled by:
  // below -89 the factor of a reference of 0 would be infinite, and their product NaN)
  const float sum = wave_sum_uniform(
      m > -INFINITY ? s * fast_exp2((m - top) * 1.4426950408889634f) : s);
  const float mine = lane_bound(m, a.groups);
  if (lane == 0) {
    part[wv] = {top, sum};
    bounds[wv] = mine;
  }
  __syncthreads();
  float bound = bounds[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) bound = fmaxf(bound, bounds[i]);
  if (m >= bound) {
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) hits |= (x[i] >= bound && inside(i) ? 1u : 0u) << i;
    while (hits != 0) {  // (few: their logits are read again)
      const int i = __builtin_ctz(hits);
      hits &= hits - 1;
      const int t = piece * kPiece + (i / kPer * kThreads + static_cast<int>(threadIdx.x)) * kPer +
                    i % kPer;
      const int n = atomicAdd(&listed, 1);
      if (n < kList) list[n] = key_of(ordered(value_of(logits[t]) + 0.f), t);
    }
  }
  __syncthreads();
  uint64_t* const out = a.keys + (static_cast<size_t>(row) * a.pieces + piece) * a.K;
  const int n = listed;
  if (n <= kList) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t mykey = list[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += list[j] > mykey ? 1 : 0;
      if (rank < a.K) out[rank] = mykey;
    }
    for (int i = n + threadIdx.x; i < a.K; i += kThreads) out[i] = 0;
  } else {
    // More equal logits than the list holds: one after another, each the largest below the
    // one before.
    uint64_t below = ~0ull;
    for (int r = 0; r < a.K; ++r) {
      uint64_t k = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint64_t o = inside(i) ? key_of(ordered(x[i] + 0.f), token(i)) : 0;
        k = o < below && o > k ? o : k;
      }
      k = wave_best(k);
      if (lane == 0) winner[r & 1][wv] = k;
      __syncthreads();
      k = winner[r & 1][0];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) k = winner[r & 1][i] > k ? winner[r & 1][i] : k;
      if (threadIdx.x == 0) out[r] = k;
      below = k;
    }
  }
  if (threadIdx.x == 0) {
    float M = -INFINITY;
    for (int i = 0; i < kWaves; ++i) M = fmaxf(M, part[i].x);
    float S = 0.f;
    for (int i = 0; i < kWaves; ++i)
      S += part[i].y *
           (part[i].x == -INFINITY ? 1.f : fast_exp2((part[i].x - M) * 1.4426950408889634f));
    a.sums[static_cast<size_t>(row) * a.pieces + piece] = {M, S};
  }
}

// A continuation, its beam and token as one number: ranked by value, then by the lower one.
struct Cand {
  double value;
  uint64_t id;
  __device__ __forceinline__ int beam() const { return static_cast<int>(id >> 32); }
  __device__ __forceinline__ int token() const { return static_cast<int>(id); }
};
__device__ __forceinline__ bool ahead(const Cand& a, const Cand& b) {
  return a.value > b.value || (a.value == b.value && a.id < b.id);
}

__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(BeamArgs a) {
  constexpr int kMergeWaves = kMergeThreads / kWave;
  constexpr int kFound = 1024;
  constexpr int kHeld = 2;  // continuations that a lane holds in registers
  __shared__ Cand found[kFound];
  __shared__ double bounds[kMergeWaves];
  // A beam's continuations are worth norm + (logit - peak), norm its score less the logarithm of
  // its sum: a peak of the largest floats would swallow the score, added to it first.
  __shared__ double norm[kMaxBeams];
  __shared__ float peak[kMaxBeams];
  __shared__ int kind[kMaxBeams];      // 0: its lists; 1: ended; 2: -inf alone
  __shared__ Cand best[kMaxBeams];
  __shared__ Cand winner[kMergeWaves];
  __shared__ int rows[kMaxBeams];      // the continuation of each row
  __shared__ int common[kMaxBeams * kMaxBeams];
  __shared__ int count;
  const int b = static_cast<int>(blockIdx.x);
  const int K = a.K;
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = uniform(threadIdx.x / kWave);
  const int per_beam = a.pieces * K;
  const int all = K * per_beam;
  const uint64_t* const lists = a.keys + static_cast<size_t>(b) * K * per_beam;
  uint64_t keys[kHeld];  // (of beams that have ended they are not written, and not used)
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    const int i = static_cast<int>(threadIdx.x) + u * kMergeThreads;
    keys[u] = i < all ? lists[i] : 0;
  }
  // (read now, for the end)
  const int ctx = a.shared != nullptr ? a.ctx[b] : 0;
  if (a.shared != nullptr) {
    for (int i = threadIdx.x; i < K * K; i += kMergeThreads)
      common[i] = a.shared[static_cast<size_t>(b) * K * K + i];
  }
  if (threadIdx.x == 0) count = 0;
  // log of a beam's sum of exponentials, a wavefront a beam
  for (int j = wv; j < K; j += kMergeWaves) {
    const int row = b * K + j;
    const float score = a.scores[row];
    const bool over = ended(a, row);
    const float2* p = a.sums + static_cast<size_t>(row) * a.pieces;
    float M = -INFINITY;
    double S = 0.;
    if (!over) {
      for (int i0 = 0; i0 < a.pieces; i0 += kWave) {
        const float2 v = i0 + lane < a.pieces ? p[i0 + lane] : float2{-INFINITY, 0.f};
        const float top = fmaxf(M, wave_max_uniform(v.x));
        S = S * (M == -INFINITY ? 1.f : fast_exp2((M - top) * 1.4426950408889634f)) +
            static_cast<double>(v.y) *
                (v.x == -INFINITY ? 1.f : fast_exp2((v.x - top) * 1.4426950408889634f));
        M = top;
      }
    }
#pragma unroll
    for (int k = 1; k < kWave; k <<= 1) S += __shfl_xor(S, k);
    if (lane == 0) {
      const double less = log(S);
      const bool whole = isfinite(score);
      kind[j] = over ? 1 : (isfinite(M) && isfinite(less) && whole ? 0 : 2);
      norm[j] = over ? (whole ? static_cast<double>(score) : -INFINITY) : score - less;
      peak[j] = M;
    }
  }
  __syncthreads();
  // continuation i of all, with its key; whether there is one
  auto cand = [&](int i, uint64_t key, Cand& c) {
    if (i >= all) return false;
    const int beam = i / per_beam;
    const int in = i - beam * per_beam;
    const int what = kind[beam];
    const int token = what == 0 ? token_of(key) : (what == 1 ? static_cast<int>(a.end_token) : in);
    c.id = static_cast<uint64_t>(beam) << 32 | static_cast<uint32_t>(token);
    c.value = what == 0 ? norm[beam] + (static_cast<double>(unordered(
                                            static_cast<uint32_t>(key >> 32))) - peak[beam])
                        : (what == 1 ? norm[beam] : -INFINITY);
    return what == 0 ? key != 0 : (what == 1 ? in == 0 : in < K && in < a.V);
  };
  // the first kHeld of this lane in registers, the others formed twice
  Cand own[kHeld];
  bool real[kHeld];
  double top = -INFINITY;
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    real[u] = cand(static_cast<int>(threadIdx.x) + u * kMergeThreads, keys[u], own[u]);
    top = real[u] && own[u].value > top ? own[u].value : top;
  }
  const int rest = static_cast<int>(threadIdx.x) + kHeld * kMergeThreads;
  for (int i = rest; i < all; i += kMergeThreads) {
    Cand c;
    if (cand(i, lists[i], c) && c.value > top) top = c.value;
  }
  const double mine = lane_bound(top, a.groups);
  if (lane == 0) bounds[wv] = mine;
  __syncthreads();
  double bound = bounds[0];
#pragma unroll
  for (int i = 1; i < kMergeWaves; ++i) bound = bounds[i] > bound ? bounds[i] : bound;
  auto list = [&](const Cand& c) {
    if (c.value < bound) return;
    const int n = atomicAdd(&count, 1);
    if (n < kFound) found[n] = c;
  };
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (real[u]) list(own[u]);
  for (int i = rest; i < all; i += kMergeThreads) {
    Cand c;
    if (cand(i, lists[i], c)) list(c);
  }
  __syncthreads();
  const int n = count;
  if (n <= kFound) {
    for (int i = threadIdx.x; i < n; i += kMergeThreads) {
      const Cand c = found[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += ahead(found[j], c) ? 1 : 0;
      if (rank < K) best[rank] = c;
    }
  } else {
    // More equal ones than the list holds: one after another.
    for (int r = 0; r < K; ++r) {
      Cand top_c = {-INFINITY, ~0ull};
      for (int i = threadIdx.x; i < all; i += kMergeThreads) {
        Cand c;
        if (cand(i, lists[i], c) && (r == 0 || ahead(best[r - 1], c)) && ahead(c, top_c))
          top_c = c;
      }
#pragma unroll
      for (int k = 1; k < kWave; k <<= 1) {
        const Cand o = {__shfl_xor(top_c.value, k),
                        __shfl_xor(static_cast<unsigned long long>(top_c.id), k)};
        top_c = ahead(o, top_c) ? o : top_c;
      }
      if (lane == 0) winner[wv] = top_c;
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int i = 1; i < kMergeWaves; ++i)
          if (ahead(winner[i], winner[0])) winner[0] = winner[i];
        best[r] = winner[0];
      }
      __syncthreads();
    }
  }
  __syncthreads();
  if (wv == 0) {  // rows of the K continuations, one a lane
    const int beam = lane < K ? best[lane].beam() : -1;
    bool stays = lane < K;
    uint32_t taken = 0;
    for (int r = 0; r < K; ++r) {
      const int p = __shfl(beam, r);  // (of all lanes: none reads one that is switched off)
      stays = stays && !(r < lane && p == beam);
      taken |= 1u << p;
    }
    const uint64_t movers = __builtin_amdgcn_ballot_w64(lane < K && !stays);
    if (lane < K) {
      int row = beam;
      if (!stays) {  // the (movers before this one)-th free row
        int left = __popcll(movers & ((1ull << lane) - 1));
        for (row = 0;; ++row) {
          if ((taken >> row & 1) == 0 && left-- == 0) break;
        }
      }
      rows[row] = lane;
    }
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < K) {
    const int j = threadIdx.x;
    const Cand c = best[rows[j]];
    const size_t at = static_cast<size_t>(b) * K + j;
    a.scores_out[at] = static_cast<float>(c.value);
    a.tokens[at] = c.token();
    a.parents[at] = c.beam();
    if (a.shared != nullptr)
      a.first[at] = c.beam() == j ? ctx : common[c.beam() * K + j];
  }
  if (a.shared == nullptr) return;
  for (int i = threadIdx.x; i < K * K; i += kMergeThreads) {
    const int p = best[rows[i / K]].beam(), q = best[rows[i % K]].beam();
    a.shared_out[static_cast<size_t>(b) * K * K + i] =
        p == q ? ctx : common[p * K + q];
  }
}

// ---- copies between beams -------------------------------------------------------
//
// Row j of a request takes the K and V of tokens [first, ctx) of the row that it goes on
// from, in every layer; rows that go on from themselves are left alone.  A workgroup copies
// blocks of (up to) 32 tokens of a kv head, K and V^T one run of memory each.  Bound by the
// bytes, each read and written once (71 MB in 8 layers: 33.9 us, the median of a trace, 4.2 TB/s
// of both); a few tokens by the launch and three dependent reads (the parents, the tables, the
// rows; 6.6 us).

constexpr int kForkThreads = 256;
constexpr int kForkLayers = 64;

struct ForkLayer {
  uint16_t* k;
  uint16_t* v;
  const int32_t* table;  // [B * K, max_pages]
  int max_pages, num_slots;
};

struct ForkArgs {
  ForkLayer layers[kForkLayers];
  const int32_t* ctx;      // [B]
  const int32_t* parents;  // [B, K]
  const int32_t* first;    // [B, K], or null: 0
  int K, NKV, D, pt_shift, vb_shift;
};

__global__ __launch_bounds__(kForkThreads) void fork_kernel(ForkArgs a) {
  const int row = static_cast<int>(blockIdx.y);
  const int b = row / a.K;
  const int parent = a.parents[row];
  const int j = row - b * a.K;
  if (parent == j || static_cast<unsigned>(parent) >= static_cast<unsigned>(a.K)) return;
  const ForkLayer& l = a.layers[blockIdx.z];
  const int cap = l.max_pages << a.pt_shift;
  int n = a.ctx[b];
  n = n < cap ? n : cap;
  int f = a.first != nullptr ? a.first[row] : 0;
  f = f > 0 ? f : 0;
  if (f >= n) return;
  const int VB = 1 << a.vb_shift;
  const int blk0 = f >> a.vb_shift;
  const int blocks = ((n - 1) >> a.vb_shift) + 1 - blk0;
  const int sub_shift = a.pt_shift - a.vb_shift;  // log2 of a page's blocks
  const int32_t* from = l.table + static_cast<size_t>(b * a.K + parent) * l.max_pages;
  const int32_t* to = l.table + static_cast<size_t>(row) * l.max_pages;
  const int k_chunks = a.D * VB / 8;  // 16-byte chunks of a block, K and V^T alike
  for (int task = blockIdx.x; task < blocks * a.NKV; task += gridDim.x) {
    const int bi = blk0 + task / a.NKV;
    const int h = task % a.NKV;
    const int src = from[bi >> sub_shift], dst = to[bi >> sub_shift];
    if (static_cast<unsigned>(src) >= static_cast<unsigned>(l.num_slots) ||
        static_cast<unsigned>(dst) >= static_cast<unsigned>(l.num_slots) || src == dst)
      continue;
    const int in = bi & ((1 << sub_shift) - 1);
    const size_t block = static_cast<size_t>(a.D) << a.vb_shift;
    const size_t s = (((static_cast<size_t>(src) * a.NKV + h) << sub_shift) + in) * block;
    const size_t d = (((static_cast<size_t>(dst) * a.NKV + h) << sub_shift) + in) * block;
    // tokens t0 .. t1 of the block
    const int t0 = f - (bi << a.vb_shift) > 0 ? f - (bi << a.vb_shift) : 0;
    const int left = n - (bi << a.vb_shift);
    const int t1 = left < VB ? left : VB;
    for (int c = threadIdx.x; c < k_chunks; c += kForkThreads) {
      const int tk = 8 * c / a.D;             // K: the token of chunk c
      const int tv = 8 * c & (VB - 1);        // V^T: its first token
      const bool k_in = tk >= t0 && tk < t1;
      const bool v_in = tv + 8 > t0 && tv < t1;
      u32x4 kk, vv;
      if (k_in) kk = *reinterpret_cast<const u32x4*>(l.k + s + 8 * c);
      if (v_in) vv = *reinterpret_cast<const u32x4*>(l.v + s + 8 * c);
      if (k_in) *reinterpret_cast<u32x4*>(l.k + d + 8 * c) = kk;
      if (v_in && tv >= t0 && tv + 8 <= t1) {
        *reinterpret_cast<u32x4*>(l.v + d + 8 * c) = vv;
      } else if (v_in) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (tv + e >= t0 && tv + e < t1)
            l.v[d + 8 * c + e] = static_cast<uint16_t>(vv[e >> 1] >> 16 * (e & 1));
      }
    }
  }
}

// Logits of a lane: 32 where the pieces then fill the card, else 8, since with few pieces the
// time is what a lane does one after another (4 beams of 49,152 tokens: 11.3 us with 8, 17.5
// with 32, both launches).
int each_of(int batch, int beams, int vocab) {
  const long long pieces = static_cast<long long>(batch) * beams * (vocab / (kThreads * 32) + 1);
  return pieces >= device_cu_count() ? 32 : 8;
}
int pieces_of(int batch, int beams, int vocab) {
  const int piece = kThreads * each_of(batch, beams, vocab);
  return (vocab + piece - 1) / piece;
}

bool beam_shape_ok(int batch, int beams, int vocab) {
  return batch > 0 && batch <= 65535 && beams > 0 && beams <= kMaxBeams && vocab > 0 &&
         vocab <= (1 << 24);
}

}  // namespace
}  // namespace voom

using namespace voom;

extern "C" size_t voom_beam_select_workspace_bytes(int batch, int beams, int vocab) {
  if (!beam_shape_ok(batch, beams, vocab)) return 0;
  const size_t rows = static_cast<size_t>(batch) * beams;
  return rows * pieces_of(batch, beams, vocab) * (beams * sizeof(uint64_t) + sizeof(float2));
}

extern "C" int voom_beam_select(const void* logits, int dtype, const float* scores,
                                const int64_t* last, int64_t end_token, const int32_t* shared,
                                const int32_t* ctx_lens, float* scores_out, int64_t* tokens,
                                int32_t* parents, int32_t* first, int32_t* shared_out,
                                void* workspace, size_t ws_bytes, int batch, int beams, int vocab,
                                hipStream_t stream) {
  const char* who = "beam_select";
  VOOM_REQUIRE(logits && scores && scores_out && tokens && parents && workspace,
               "%s: null pointer argument", who);
  VOOM_REQUIRE(beam_shape_ok(batch, beams, vocab),
               "%s: %d requests of %d beams (at most %d) over %d tokens", who, batch, beams,
               kMaxBeams, vocab);
  VOOM_REQUIRE(dtype == VOOM_DTYPE_BF16 || dtype == VOOM_DTYPE_F32,
               "%s: logits must be bf16 or fp32", who);
  VOOM_REQUIRE(last == nullptr || (end_token >= 0 && end_token < vocab),
               "%s: the end token must be one of the %d", who, vocab);
  VOOM_REQUIRE(shared == nullptr || (ctx_lens && first && shared_out && shared != shared_out),
               "%s: shared needs ctx_lens, first and another shared_out", who);
  VOOM_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == VOOM_DTYPE_BF16 ? 2 : 4) == 0 &&
                   reinterpret_cast<uintptr_t>(workspace) % 8 == 0,
               "%s: logits and workspace must be aligned", who);
  VOOM_REQUIRE(ws_bytes >= voom_beam_select_workspace_bytes(batch, beams, vocab),
               "%s: workspace %zu bytes < required %zu", who, ws_bytes,
               voom_beam_select_workspace_bytes(batch, beams, vocab));
  BeamArgs a;
  a.logits = logits;
  a.scores = scores;
  a.last = last;
  a.end_token = end_token;
  a.shared = shared;
  a.ctx = ctx_lens;
  a.scores_out = scores_out;
  a.tokens = tokens;
  a.parents = parents;
  a.first = first;
  a.shared_out = shared_out;
  a.B = batch;
  a.K = beams;
  a.V = vocab;
  a.pieces = pieces_of(batch, beams, vocab);
  a.groups = 1 << ilog2(beams);
  a.keys = static_cast<uint64_t*>(workspace);
  a.sums = reinterpret_cast<float2*>(a.keys + static_cast<size_t>(batch) * beams * a.pieces *
                                                  beams);
  const dim3 grid(static_cast<unsigned>(a.pieces), static_cast<unsigned>(batch),
                  static_cast<unsigned>(beams));
  const bool many = each_of(batch, beams, vocab) == 32;
  if (dtype == VOOM_DTYPE_BF16 && many)
    hipLaunchKernelGGL((beam_pieces_kernel<uint16_t, 32>), grid, dim3(kThreads), 0, stream, a);
  else if (dtype == VOOM_DTYPE_BF16)
    hipLaunchKernelGGL((beam_pieces_kernel<uint16_t, 8>), grid, dim3(kThreads), 0, stream, a);
  else if (many)
    hipLaunchKernelGGL((beam_pieces_kernel<float, 32>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((beam_pieces_kernel<float, 8>), grid, dim3(kThreads), 0, stream, a);
  const int rc = VOOM_LAUNCH_CHECK("beam_select: pieces launch");
  if (rc) return rc;
  hipLaunchKernelGGL(beam_merge_kernel, dim3(static_cast<unsigned>(batch)), dim3(kMergeThreads),
                     0, stream, a);
  return VOOM_LAUNCH_CHECK("beam_select: merge launch");
}

extern "C" int voom_fork_kv(void* const* k_pools, void* const* v_pools,
                            const int32_t* const* block_tables, const int* max_pages,
                            const int* num_slots, int num_layers, const int32_t* ctx_lens,
                            const int32_t* parents, const int32_t* first, int batch, int beams,
                            int num_kv_heads, int head_dim, int page_tokens, hipStream_t stream) {
  const char* who = "fork_kv";
  VOOM_REQUIRE(k_pools && v_pools && block_tables && max_pages && num_slots && ctx_lens && parents,
               "%s: null pointer argument", who);
  VOOM_REQUIRE(num_layers > 0 && batch > 0 && beams > 0 && num_kv_heads > 0 &&
                   static_cast<long long>(batch) * beams <= 65535,
               "%s: bad geometry (%d layers, batch %d, %d beams, %d kv heads)", who, num_layers,
               batch, beams, num_kv_heads);
  VOOM_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= 1024,
               "%s: head_dim %d must be a multiple of 8 up to 1024", who, head_dim);
  VOOM_REQUIRE(is_pow2(page_tokens) && page_tokens >= 8 && page_tokens <= 4096,
               "%s: page_tokens %d must be a power of two in [8, 4096]", who, page_tokens);
  for (int i = 0; i < num_layers; ++i) {
    VOOM_REQUIRE(k_pools[i] && v_pools[i] && block_tables[i] &&
                     reinterpret_cast<uintptr_t>(k_pools[i]) % 16 == 0 &&
                     reinterpret_cast<uintptr_t>(v_pools[i]) % 16 == 0,
                 "%s: pools must be 16-byte aligned", who);
    VOOM_REQUIRE(num_slots[i] > 0 && max_pages[i] > 0 &&
                     static_cast<long long>(max_pages[i]) * page_tokens < (1LL << 30),
                 "%s: layer %d has %d pages of a pool of %d", who, i, max_pages[i], num_slots[i]);
  }
  ForkArgs a;
  a.ctx = ctx_lens;
  a.parents = parents;
  a.first = first;
  a.K = beams;
  a.NKV = num_kv_heads;
  a.D = head_dim;
  a.pt_shift = ilog2(page_tokens);
  a.vb_shift = a.pt_shift < 5 ? a.pt_shift : 5;
  for (int l0 = 0; l0 < num_layers; l0 += kForkLayers) {
    const int layers = num_layers - l0 < kForkLayers ? num_layers - l0 : kForkLayers;
    long long most = 1;  // blocks that a row can hold
    for (int i = 0; i < layers; ++i) {
      a.layers[i] = {static_cast<uint16_t*>(k_pools[l0 + i]),
                     static_cast<uint16_t*>(v_pools[l0 + i]), block_tables[l0 + i],
                     max_pages[l0 + i], num_slots[l0 + i]};
      const long long blocks = static_cast<long long>(max_pages[l0 + i])
                               << (a.pt_shift - a.vb_shift);
      most = blocks > most ? blocks : most;
    }
    // Workgroups of a (row, layer): as many as give the card 32 each, few enough to launch
    // fast where most of the rows stay.
    const long long rows = static_cast<long long>(batch) * beams * layers;
    long long each = (32LL * device_cu_count() + rows - 1) / rows;
    if (each > most * num_kv_heads) each = most * num_kv_heads;
    hipLaunchKernelGGL(fork_kernel,
                       dim3(static_cast<unsigned>(each), static_cast<unsigned>(batch * beams),
                            static_cast<unsigned>(layers)),
                       dim3(kForkThreads), 0, stream, a);
    const int rc = VOOM_LAUNCH_CHECK("fork_kv: launch");
    if (rc) return rc;
  }
  return VOOM_OK;
}
