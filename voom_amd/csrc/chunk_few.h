// What the kernels of single tokens and short chunks share (gqa_chunk.hip,
// gqa_chunk_token.hip): units of work, a row's view of the cache, the softmax of a block and
// the merge of cut segments.
#pragma once

#include "chunk_rows.h"
#include "paged_rows.h"

namespace voom {

// How a kernel takes a call: row tiles of kRows, stages of kTok tokens, kLead units that
// stand for what a segment costs besides its stages, and kLeast units of a worker, since each
// leaves pieces to be merged.
template <int ROWS, int TOK, int LEAD, int LEAST>
struct Geometry {
  static constexpr int kRows = ROWS, kTok = TOK, kLead = LEAD, kLeast = LEAST;
};

// U units over W workers, or fewer.
template <class Geo>
__device__ __forceinline__ Split split_of(int U, int W) {
  const int most = U / Geo::kLeast;
  return Split(U, most < W ? (most > 1 ? most : 1) : W);
}

// Units of a sequence: for every kv head and row tile the stages that its rows see, after
// kLead units.  Stages from `pre` on lie `gap` further on in the context.
template <class Geo>
struct Units {
  int chunks, tiles, pre, gap;
  __device__ __forceinline__ int all(const ChunkArgs& a) const {
    if (a.W == 0) return tiles * a.NKV;
    return chunks == 0 ? 0 : (chunks + Geo::kLead) * tiles * a.NKV;
  }
  __device__ __forceinline__ Units(const ChunkArgs& a, int b) {
    constexpr int kTok = Geo::kTok, kRows = Geo::kRows;
    int base;
    const int ctx = context_of(a, b), n = new_of(a, b, base), p = prefix_of(a, b, ctx);
    const Sight first(a, ctx, n, p, 0);
    pre = (p + kTok - 1) / kTok;
    gap = first.lo / kTok - pre;
    gap = gap < 0 ? 0 : gap;
    chunks = n == 0 ? 0 : (ctx + kTok - 1) / kTok - gap;
    // (rows behind a padded sequence's are written by its segments where none is cut)
    tiles = ((a.W == 0 && a.starts == nullptr ? a.T : n) * a.G + kRows - 1) / kRows;
  }
};

// The units of up to 64 sequences from `base` on, one per lane, and their inclusive sum.
template <class Geo>
__device__ __forceinline__ Units<Geo> scan_units(const ChunkArgs& a, int base, int lane, int& x) {
  const bool in = base + lane < a.B;
  const Units<Geo> u(a, in ? base + lane : 0);
  x = wave_inclusive_scan(in ? u.all(a) : 0, lane);
  return u;
}

// What the row of this lane's column sees, and its score's slope.
struct View {
  int ctx, pre, at, lo, hi;
  float slope;  // log2 units
  bool biased;
  // Bit e: it sees token pos + e, e < 8.
  __device__ __forceinline__ uint32_t seen(int pos) const {
    return hi > 0 ? bits_in(pos, lo, hi) | bits_in(pos, 0, pre) : 0u;
  }
};

// Scores in log2 units, of this lane's 8 tokens from pos on.
__device__ __forceinline__ void score(f32x4 (&sc)[1][2], const ChunkArgs& a, const View& view,
                                      int pos) {
  if (a.cap != 0.f) {
    float x[8];
    bool far = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = sc[0][e >> 2][e & 3] * a.cap_k;
      far |= fabsf(x[e]) > kNear;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sc[0][e >> 2][e & 3] = a.cap * x[e] * tanh_ratio(x[e] * x[e]);
    if (__builtin_amdgcn_ballot_w64(far) != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = capped_far(x[e], a.cap);
        sc[0][e >> 2][e & 3] = fabsf(x[e]) > kNear ? y : sc[0][e >> 2][e & 3];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) sc[0][e >> 2][e & 3] *= a.scale;
  }
  if (view.biased) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = view.at - (pos + e);
      sc[0][e >> 2][e & 3] -= view.slope * static_cast<float>(d < 0 ? -d : d);
    }
  }
}

// Forms P of a block's scores.
template <int D>
__device__ __forceinline__ void weights_of(const f32x4 (&sc)[1][2], State<D, 1>& st,
                                           u32x4 (&p)[1]) {
  float mx[1] = {fmaxf(sc[0][0][0], sc[0][1][0])};
#pragma unroll
  for (int e = 1; e < 4; ++e) mx[0] = fmaxf(fmaxf(mx[0], sc[0][0][e]), sc[0][1][e]);
  if (__builtin_amdgcn_ballot_w64(mx[0] > st.m[0] + kSlack) != 0) raise_maxima<D, 1>(mx, st);
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = fast_exp2(sc[0][e >> 2][e & 3] - st.m[0]);
  st.l[0] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
  for (int e = 0; e < 4; ++e) p[0][e] = pack_bf16x2(w[2 * e], w[2 * e + 1]);
}

constexpr int kReduceWaves = 4;

// One wavefront per row: merges the pieces of its segment, where the split cut it, and
// writes the rows that no segment holds.
template <int D, class Geo>
__global__ __launch_bounds__(kReduceWaves * kWave) void gqa_chunk_reduce_kernel(ChunkArgs a) {
  constexpr int kRows = Geo::kRows, kLead = Geo::kLead;
  // A wavefront holds the row of kTogether pieces at a time, 4 dims per lane.
  constexpr int kLanes = D / 4;
  constexpr int kTogether = kWave / kLanes;
  constexpr int kAhead = 8;  // loads in flight
  const int lane = threadIdx.x & (kWave - 1);
  const int kvh = static_cast<int>(blockIdx.y);
  const int all = static_cast<int>(blockIdx.x) * kReduceWaves + uniform(threadIdx.x / kWave);
  int b = static_cast<int>(blockIdx.z);
  int rr = all;  // the row within its sequence
  if (a.starts != nullptr) {
    const int token = all / a.G;
    if (token >= a.N) return;
    // the last sequence that starts at or before the token (those behind it are empty)
    b = -1;
    for (int at = 0; at < a.B; at += kWave) {
      const bool in = at + lane < a.B && a.starts[at + lane < a.B ? at + lane : 0] <= token;
      b += __popcll(__builtin_amdgcn_ballot_w64(in));
    }
    if (b < 0) return;
  } else if (all >= a.T * a.G) {
    return;
  }
  int base;
  const int n = uniform(new_of(a, b, base));
  if (a.starts != nullptr) rr -= base * a.G;
  const int t = rr / a.G;
  if (a.starts != nullptr && (t < 0 || t >= n)) return;  // of no sequence
  const int tile = rr / kRows;
  const int r = rr - tile * kRows;
  const int head = kvh * a.G + (rr - t * a.G);
  const size_t at = out_at(a, b, base, t, head);
  const int sub = lane / kLanes;
  const int dim = lane % kLanes * 4;
  int first = 0, last = -1;
  if (t < n) {  // (else 0)
    // units before sequence b, and of all; stages and row tiles of b
    int before = 0, chunks = 0, tiles = 1, U = 0;
    for (int from = 0; from < a.B; from += kWave) {
      int x;
      const Units<Geo> units = scan_units<Geo>(a, from, lane, x);
      if (b >= from && b < from + kWave) {
        chunks = __builtin_amdgcn_readlane(units.chunks, b - from);
        tiles = __builtin_amdgcn_readlane(units.tiles, b - from);
        before = U + __builtin_amdgcn_readlane(x, b - from) - (chunks + kLead) * tiles * a.NKV;
      }
      U += __builtin_amdgcn_readlane(x, kWave - 1);
    }
    if (chunks != 0) {  // (a context of no tokens has no segments)
      const Split split = split_of<Geo>(U, a.W);
      const int S = before + (kvh * tiles + tile) * (chunks + kLead) + kLead;
      first = split.group(S);
      last = split.group(S + chunks - 1);
      if (first == last) return;  // written by its workgroup
    }
  }
  // Up to 64 pieces at a time, one per lane for their maxima and sums.  A workgroup leaves
  // the piece that starts a segment, its last one, in its second slot.
  float M = -FLT_MAX, L = 0.f;
  f32x4 acc = {};
  for (int w0 = first; w0 <= last; w0 += kWave) {
    const int m = last - w0 + 1 < kWave ? last - w0 + 1 : kWave;
    const size_t p0 = 2 * static_cast<size_t>(w0) * kRows + r;
    const int odd = w0 == first ? kRows : 0;  // of the first one
    auto row_at = [&](int k) {
      k = k < m ? k : m - 1;
      return p0 + 2 * static_cast<size_t>(k) * kRows + (k == 0 ? odd : 0);
    };
    f32x4 v[kAhead];
    auto read = [&](int k0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        v[u] = *reinterpret_cast<const f32x4*>(a.part_o + row_at(k0 + u * kTogether + sub) * D +
                                               dim);
    };
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + row_at(lane) * 2);
    read(0);  // (under way while the weights are formed)
    const float mn = fmaxf(M, wave_max_uniform(lane < m ? ml.x : -FLT_MAX));
    const float wt = lane < m ? fast_exp2(ml.x - mn) : 0.f;
    const float f = fast_exp2(M - mn);
    M = mn;
    L = L * f + wave_sum_uniform(lane < m ? ml.y * wt : 0.f);
    acc *= f;
    for (int k0 = 0; k0 < m; k0 += kAhead * kTogether) {
      if (k0 != 0) read(k0);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u * kTogether + sub;
        const float ws = __shfl(wt, k & (kWave - 1));
        if (k < m) acc += v[u] * ws;  // (0 times the infinity of a piece read again is NaN)
      }
    }
  }
#pragma unroll
  for (int k = kLanes; k < kWave; k <<= 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], k);
  }
  const bool empty = L == 0.f;
  const float inv = 1.f / L;
  if (sub == 0)
    *reinterpret_cast<u32x2*>(a.out + at * D + dim) =
        empty ? u32x2{0u, 0u}
              : u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv),
                      pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  if (a.lse != nullptr && lane == 0)
    a.lse[at] = empty ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
}

// The reduce launch behind a split call.
template <int D, class Geo>
int launch_reduce(const ChunkArgs& a, hipStream_t stream) {
  const bool packed = a.starts != nullptr;
  const long long rows = static_cast<long long>(packed ? a.N : a.T) * a.G;
  const dim3 grid(static_cast<unsigned>((rows + kReduceWaves - 1) / kReduceWaves),
                  static_cast<unsigned>(a.NKV), static_cast<unsigned>(packed ? 1 : a.B));
  hipLaunchKernelGGL((gqa_chunk_reduce_kernel<D, Geo>), grid, dim3(kReduceWaves * kWave), 0,
                     stream, a);
  return VOOM_LAUNCH_CHECK("paged_gqa_chunk: reduce launch");
}

}  // namespace voom
