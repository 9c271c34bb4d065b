// Paged GQA attention of drafted tokens for gfx950: the verify step of
// speculative decoding over the paged K/V cache.
//
// Sequence b holds ctx[b] tokens; the newest n = lens[b] of them are drafts,
// their K/V already in the cache.  Draft t sees the ctx - n tokens before the
// drafts and those drafts j whose mask[t][j] is set (its ancestors and itself in
// a tree; j <= t without a mask):
//   out[t][h] = sum_p softmax_p(scale q[t][h] . k[p]) v[p],  lse = log sum_p exp.
// Rows t >= n, and rows that see nothing, give 0 and -inf.
//
// What bounds it: K and V of the context once (4 D bytes per token and kv head)
// until about 100 (draft, head of a group) rows share them, then matrix work,
// 4 NQ D flops per (draft, visible key).
//
// Work decomposition.  The rows of one (sequence, kv head) go in tiles of 16 NT
// (NT = 1, 2, 4) that share every K/V byte.  A unit is a chunk of 128 tokens of one
// (sequence, kv head, row tile) segment, 32 per wavefront; the units of all segments
// lie end to end and workgroup w of W takes [w U/W, (w+1) U/W), so that all stream
// the same number of bytes whatever the context lengths.  The wavefronts of a
// workgroup merge their states through LDS.  A segment within one workgroup is
// written from there; of the others a workgroup holds at most two pieces (its first
// and its last), which gqa_tree_reduce_kernel merges.
//
// A wavefront has two buffers of 32 tokens of K and V^T in LDS of its own, filled by
// direct-to-LDS loads (1 KiB each), so that one block is under way while the other is
// computed, without a barrier.  The row tiles are in the N dimension:
//   scores^T[token][row] = K . Q^T,  out^T[dim][row] += V^T . P^T   16x16x32 bf16
// Row 4g + r of score tile t holds token 8g + 4t + r, so that a lane's scores are
// the 8 consecutive tokens that its P^T operand needs.  (Blocks in registers instead, as
// in the decode kernel, leave too few for 64 rows: 116 spilled, 1,076 us where this takes
// 371.)
//
// P is rounded to bf16 for the matrix units; its sum, and with it the LSE, is kept
// of the unrounded fp32 weights (the roundings average out in the output, whose own
// rounding is as large as one of them).
#include "common.h"

#include <cfloat>
#include <cmath>

namespace voom {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kBlk = 32;               // tokens of a K/V block in the pool
constexpr int kChunk = kWaves * kBlk;  // tokens of a unit
constexpr int kMaxBatch = 1024;
constexpr int kMaxDrafts = 1024;

struct TreeArgs {
  const uint16_t* q;      // [B, NQ, T, D]
  const uint16_t* k_pool;
  const uint16_t* v_pool;
  const int32_t* table;   // [B, max_pages]
  const int32_t* ctx;     // [B]
  const int32_t* lens;    // [B], or null: T each
  const uint8_t* mask;    // [T, T] or [B, T, T] of 0 / 1, or null: causal
  uint16_t* out;          // [B, T, NQ, D]
  float* lse;             // [B, T, NQ], or null
  float* part_o;          // [2 W, 16 NT, D]
  float* part_ml;         // [2 W, 16 NT, 2]
  long long mask_stride;  // elements from one sequence's mask to the next
  int B, NQ, NKV, G, T, max_pages, pt_shift, num_slots;
  int R;         // rows of a (sequence, kv head): T * G, (draft, head), head fastest
  int tiles;     // row tiles along R
  int W;         // workgroups of the split, 0: one per segment
  int per_xcd;   // workgroups per XCD
  // |softmax scale| in log2 units, > 0.  The sign is applied to q (q_flip =
  // 0x80008000), a scale of 0 by clearing q but for infinities and NaN (q_zero,
  // scale 1).
  float scale;
  uint32_t q_flip;
  bool q_zero;
};

__device__ __forceinline__ int context_of(const TreeArgs& a, int b) {
  const int cap = a.max_pages << a.pt_shift;
  const int c = a.ctx[b];
  return c < 0 ? 0 : (c > cap ? cap : c);
}

__device__ __forceinline__ int drafts_of(const TreeArgs& a, int b, int ctx) {
  int n = a.lens != nullptr ? a.lens[b] : a.T;
  n = n < 0 ? 0 : (n > a.T ? a.T : n);
  return n < ctx ? n : ctx;
}

__device__ __forceinline__ int chunks_of(int ctx) { return (ctx + kChunk - 1) / kChunk; }

// Workgroup of the split that holds unit u (the last w with w U/W <= u).
__device__ __forceinline__ long long group_of_unit(long long u, long long U, int W) {
  return ((u + 1) * W - 1) / U;
}

typedef __attribute__((address_space(3))) void lds_void;

// Chunk c (16 bytes) of K row r sits at c ^ k_swizzle(r) of its row, chunk c of V^T row
// d at c ^ (d >> 2 & 3): the 16 rows of an operand read then spread over all banks.
template <int D>
__device__ __forceinline__ int k_swizzle(int r) {
  return D == 128 ? (r & 3) | ((r >> 3) & 3) << 2 : ((r >> 1) & 1) | ((r >> 3) & 3) << 1;
}

// The keys of the pages that one segment's wavefront walks.
struct Pages {
  const int32_t* row;  // the sequence's table row
  int kvh, base, tab;  // base: first of the 64 pages whose slots the lanes hold in tab
};

constexpr int kTileElems(int D) { return 2 * kBlk * D; }  // K block, V^T block

// Starts the loads of block bi into a wavefront's buffer.
template <int D, int AUX>
__device__ __forceinline__ void load_tile(uint16_t* tile, const TreeArgs& a, Pages& pg, int bi,
                                          int lane) {
  constexpr int kPieces = kBlk * D / 512;  // 1 KiB loads per block
  constexpr int kCpr = D / 8;              // 16-byte chunks of a K row
  const int sub_shift = a.pt_shift - 5;
  const int page = bi >> sub_shift;
  const int sub = bi & ((1 << sub_shift) - 1);
  if (page >= pg.base + kWave) {
    pg.base = page;
    const int p = page + lane;
    pg.tab = p < a.max_pages ? pg.row[p] : 0;
    wait_vmem_all();  // here, not at the readlane below on every block
  }
  int slot = __builtin_amdgcn_readlane(pg.tab, page - pg.base);
  if (static_cast<unsigned>(slot) >= static_cast<unsigned>(a.num_slots)) slot = 0;
  const size_t at = ((static_cast<size_t>(slot) * a.NKV + pg.kvh) << sub_shift) + sub;
  const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(a.k_pool + at * (kBlk * D)), static_cast<short>(0), kBlk * D * 2,
      0x00020000);
  const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(a.v_pool + at * (kBlk * D)), static_cast<short>(0), kBlk * D * 2,
      0x00020000);
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int r = i * (kWave / kCpr) + lane / kCpr;
    const int src = r * (D * 2) + 16 * ((lane % kCpr) ^ k_swizzle<D>(r));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(kr, (lds_void*)(tile + i * 512), 16, src, 0, 0, AUX);
  }
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int src = (lane >> 2) * (kBlk * 2) + 16 * ((lane & 3) ^ ((lane >> 4) & 3));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(vr, (lds_void*)(tile + kBlk * D + i * 512), 16, src,
                                             i * 1024, 0, AUX);
  }
}

// K operand of score tile t, k-step s, and V^T operand of dims 16 n.. of a buffer.
template <int D>
__device__ __forceinline__ u32x4 read_k(const uint16_t* tile, int t, int s, int lane) {
  const int i16 = lane & 15, g = lane >> 4;
  const int r = 8 * (i16 >> 2) + (i16 & 3) + 4 * t;
  return *reinterpret_cast<const u32x4*>(tile + r * D + 8 * ((4 * s + g) ^ k_swizzle<D>(r)));
}
template <int D>
__device__ __forceinline__ u32x4 read_v(const uint16_t* tile, int n, int lane) {
  const int i16 = lane & 15, g = lane >> 4;
  return *reinterpret_cast<const u32x4*>(tile + kBlk * D + (16 * n + i16) * kBlk +
                                         8 * (g ^ (i16 >> 2)));
}

template <int D, int NT>
struct State {
  f32x4 acc[NT][D / 16];
  float m[NT];  // reference maximum, log2 units, the same in all lanes of a column
  float l[NT];  // sum of this lane's weights
};

// Which keys the rows of this lane's columns see.
template <int NT>
struct View {
  int ctx, prefix, drafts;
  int t[NT];            // the draft of the column's row in each tile; T: no row
  const uint8_t* mask;  // the sequence's mask, or null
  int T;
  // Bit e: the row of tile i sees token pos + e.  Straight-line code: every mask
  // byte is loaded from inside the mask and then chosen or not.
  template <int N>
  __device__ __forceinline__ uint32_t seen(int i, int pos) const {
    const int row = t[i] < T ? t[i] : T - 1;
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int j = pos + e - prefix;
      int ok = j <= t[i];
      if (mask != nullptr) {
        const int jc = j < 0 ? 0 : (j < T ? j : T - 1);
        ok = mask[static_cast<size_t>(row) * T + jc] != 0;
      }
      ok = (j < 0) | ((j < drafts) & ok);
      bits |= static_cast<uint32_t>(ok) << e;
    }
    return t[i] < drafts ? bits : 0u;
  }
};

template <int D, int NT>
__device__ __forceinline__ void scores_of(const uint16_t* tile, const uint16_t* ql,
                                          f32x4 (&sc)[NT][2], int lane) {
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    sc[i][0] = f32x4{};
    sc[i][1] = f32x4{};
  }
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    const u32x4 k0 = read_k<D>(tile, 0, s, lane), k1 = read_k<D>(tile, 1, s, lane);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const u32x4 q = *reinterpret_cast<const u32x4*>(ql + i * 16 * (D + 8) + 32 * s);
      sc[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k0),
                                                         __builtin_bit_cast(bf16x8, q), sc[i][0],
                                                         0, 0, 0);
      sc[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k1),
                                                         __builtin_bit_cast(bf16x8, q), sc[i][1],
                                                         0, 0, 0);
    }
  }
}

// Raises the reference maxima to those of the scores, and forms P.
template <int D, int NT>
__device__ __forceinline__ void weights_of(const f32x4 (&sc)[NT][2], float scale,
                                           State<D, NT>& st, u32x4 (&p)[NT]) {
  float mx[NT];
  bool up = false;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float x = fmaxf(sc[i][0][0], sc[i][1][0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) x = fmaxf(fmaxf(x, sc[i][0][e]), sc[i][1][e]);
    mx[i] = x * scale;
    up |= mx[i] > st.m[i];
  }
  if (__builtin_amdgcn_ballot_w64(up) != 0) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float mn = fmaxf(st.m[i], wave_max_across_groups(mx[i]));
      float alpha = fast_exp2(st.m[i] - mn);
      asm volatile("" : "+v"(alpha));  // keeps the rescaling inside the branch
      st.m[i] = mn;
      st.l[i] *= alpha;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) st.acc[i][n] *= alpha;
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[e] = fast_exp2(__builtin_fmaf(sc[i][e >> 2][e & 3], scale, -st.m[i]));
    st.l[i] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
    for (int e = 0; e < 4; ++e) p[i][e] = pack_bf16x2(w[2 * e], w[2 * e + 1]);
  }
}

template <int D, int NT>
__device__ __forceinline__ void whole_block(const uint16_t* tile, const uint16_t* ql, float scale,
                                            State<D, NT>& st, int lane) {
  f32x4 sc[NT][2];
  u32x4 p[NT];
  scores_of<D, NT>(tile, ql, sc, lane);
  weights_of<D, NT>(sc, scale, st, p);
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    const u32x4 v = read_v<D>(tile, n, lane);
#pragma unroll
    for (int i = 0; i < NT; ++i)
      st.acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v),
                                                             __builtin_bit_cast(bf16x8, p[i]),
                                                             st.acc[i][n], 0, 0, 0);
  }
}

// A block with drafts or with tokens past the end.  Keys that a row does not see
// score -inf.  Tokens past the end are garbage and are cut out of V^T; a draft that
// only some rows see has P = 0 in the others, but 0 times a NaN or an infinity is
// NaN: where V holds one it is taken out, and products of indicators (V is NaN, +inf,
// -inf; the row sees the key) say which sums it belongs to.
template <int D, int NT>
__device__ __forceinline__ void edge_block(const uint16_t* tile, const uint16_t* ql, float scale,
                                           State<D, NT>& st, const View<NT>& view, int bi,
                                           int lane) {
  const int g = lane >> 4;
  f32x4 sc[NT][2];
  u32x4 p[NT];
  scores_of<D, NT>(tile, ql, sc, lane);
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const uint32_t seen = view.template seen<8>(i, bi * kBlk + 8 * g);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sc[i][e >> 2][e & 3] = (seen >> e & 1) != 0 ? sc[i][e >> 2][e & 3] : -INFINITY;
  }
  weights_of<D, NT>(sc, scale, st, p);
  const int valid = view.ctx - bi * kBlk - 8 * g;
  uint32_t keep[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    keep[e] = (2 * e < valid ? 0xffffu : 0u) | (2 * e + 1 < valid ? 0xffff0000u : 0u);
  uint32_t odd = 0;  // not 0: V holds a NaN or an infinity
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    u32x4 v = read_v<D>(tile, n, lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t bad = nan_bf16(v[e] & keep[e]);
      odd |= bad;
      v[e] &= keep[e] & ~bad;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
      st.acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v),
                                                             __builtin_bit_cast(bf16x8, p[i]),
                                                             st.acc[i][n], 0, 0, 0);
  }
  if (__builtin_amdgcn_ballot_w64(odd != 0) == 0) return;
  u32x4 ones[NT];  // 1 where the row sees the key
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const uint32_t seen = view.template seen<8>(i, bi * kBlk + 8 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      ones[i][e] = ((seen >> 2 * e & 1) != 0 ? 0x3f80u : 0u) |
                   ((seen >> (2 * e + 1) & 1) != 0 ? 0x3f800000u : 0u);
  }
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    const u32x4 v = read_v<D>(tile, n, lane);
    u32x4 is_nan, is_pos, is_neg;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = v[e] & keep[e], lo = x & 0xffffu, hi = x >> 16;
      is_nan[e] = ((lo & 0x7fffu) > 0x7f80u ? 0x3f80u : 0u) |
                  ((hi & 0x7fffu) > 0x7f80u ? 0x3f800000u : 0u);
      is_pos[e] = (lo == 0x7f80u ? 0x3f80u : 0u) | (hi == 0x7f80u ? 0x3f800000u : 0u);
      is_neg[e] = (lo == 0xff80u ? 0x3f80u : 0u) | (hi == 0xff80u ? 0x3f800000u : 0u);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const auto count = [&](u32x4 x) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x),
                                                       __builtin_bit_cast(bf16x8, ones[i]),
                                                       f32x4{}, 0, 0, 0);
      };
      const f32x4 nan = count(is_nan), pos = count(is_pos), neg = count(is_neg);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float add = nan[e] > 0.f ? NAN : 0.f;
        add += pos[e] > 0.f ? INFINITY : 0.f;
        add -= neg[e] > 0.f ? INFINITY : 0.f;
        st.acc[i][n][e] += add;
      }
      __builtin_amdgcn_sched_barrier(0);  // one set of products in registers at a time
    }
  }
}

// Exclusive prefix sum of the sequences' chunk counts into seg[0..B]; ends with a
// barrier.
__device__ void chunk_prefix(const TreeArgs& a, int* seg, int* wave_tot) {
  const int t = threadIdx.x;
  const int lane = t & (kWave - 1);
  const int wv = t / kWave;
  int carry = 0;
  for (int base = 0; base < a.B; base += kThreads) {
    const int i = base + t;
    const int n = i < a.B ? chunks_of(context_of(a, i)) : 0;
    const int x = wave_inclusive_scan(n, lane);
    if (lane == kWave - 1) wave_tot[wv] = x;
    __syncthreads();
    int before = carry;
    for (int k = 0; k < wv; ++k) before += wave_tot[k];
    if (i < a.B) seg[i] = before + x - n;
    for (int k = 0; k < kWaves; ++k) carry += wave_tot[k];
    __syncthreads();
  }
  if (t == 0) seg[a.B] = carry;
  __syncthreads();
}

template <int D, int NT, int AUX>
__global__ __launch_bounds__(kThreads, D == 64 ? 2 : 1) void gqa_tree_kernel(TreeArgs a) {
  constexpr int kRows = 16 * NT;
  constexpr int kPad = D + 4;  // floats of a row in LDS: 16 rows start in 16 bank groups
  __shared__ int seg[kMaxBatch + 1];
  __shared__ int wave_tot[kWaves];
  // The wavefronts' buffers.  Two distinct objects, so that reads of one provably miss
  // the other's pending direct-to-LDS loads; the merge uses them when the loop is done.
  __shared__ __attribute__((aligned(1024))) uint16_t tile_a[kWaves][kTileElems(D)];
  __shared__ __attribute__((aligned(1024))) uint16_t tile_b[kWaves][kTileElems(D)];
  static_assert(sizeof(float) * kWaves * 16 * kPad <= sizeof(tile_a), "a merge buffer fits");
  __shared__ __attribute__((aligned(16))) uint16_t q_rows[kRows][D + 8];
  __shared__ float red_m[kWaves][kRows];
  __shared__ float red_l[kWaves][kRows];

  const int lane = threadIdx.x & (kWave - 1);
  const int wv = uniform(threadIdx.x / kWave);
  const int i16 = lane & 15;
  const int g = lane >> 4;
  // Consecutive workgroups of one XCD take consecutive units, so that the row tiles
  // that read the same keys share an L2.
  const int bid = static_cast<int>(blockIdx.x);
  const int w = (bid & 7) * a.per_xcd + (bid >> 3);

  int b, kvh, tile, c0, c1, chunks;
  long long u0 = 0, u1 = 0, begin = 0;
  int We = 0;
  const int per_b = a.NKV * a.tiles;
  if (a.W == 0) {
    if (w >= a.B * per_b) return;
    b = w / per_b;
    chunks = uniform(chunks_of(context_of(a, b)));
    const int s = w - b * per_b;
    kvh = s / a.tiles;
    tile = s - kvh * a.tiles;
  } else {
    chunk_prefix(a, seg, wave_tot);
    const long long U = static_cast<long long>(uniform(seg[a.B])) * per_b;
    We = static_cast<int>(U < a.W ? U : a.W);
    if (w >= We) return;
    u0 = static_cast<long long>(w) * U / We;
    u1 = static_cast<long long>(w + 1) * U / We;
    int lo = 0, hi = a.B - 1;  // the sequence that holds unit u0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (static_cast<long long>(uniform(seg[mid])) * per_b <= u0) lo = mid; else hi = mid - 1;
    }
    b = lo;
    chunks = uniform(seg[b + 1]) - uniform(seg[b]);
    const long long first = static_cast<long long>(uniform(seg[b])) * per_b;
    const int s = static_cast<int>((u0 - first) / chunks);
    kvh = s / a.tiles;
    tile = s - kvh * a.tiles;
    begin = first + static_cast<long long>(s) * chunks;
  }
  for (int piece = 0;; ++piece) {
    if (a.W == 0) {
      c0 = 0;
      c1 = chunks;
    } else {
      c0 = static_cast<int>(u0 - begin);
      c1 = static_cast<int>((u1 < begin + chunks ? u1 : begin + chunks) - begin);
    }
    const int ctx = uniform(context_of(a, b));
    View<NT> view;
    view.ctx = ctx;
    view.drafts = uniform(drafts_of(a, b, ctx));
    view.prefix = ctx - view.drafts;
    view.mask = a.mask != nullptr ? a.mask + a.mask_stride * b : nullptr;
    view.T = a.T;
    // the rows' queries, for all wavefronts
    for (int idx = threadIdx.x; idx < kRows * (D / 8); idx += kThreads) {
      const int row = idx / (D / 8);
      const int c = idx - row * (D / 8);
      const int r = tile * kRows + row;
      const int rc = r < a.R ? r : 0;
      const int t = rc / a.G;
      const int head = kvh * a.G + (rc - t * a.G);
      u32x4 x = *reinterpret_cast<const u32x4*>(
          a.q + ((static_cast<size_t>(b) * a.NQ + head) * a.T + t) * D + 8 * c);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] ^= a.q_flip;
        if (a.q_zero) x[e] = nan_bf16(x[e]);
      }
      *reinterpret_cast<u32x4*>(&q_rows[row][8 * c]) = x;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = tile * kRows + 16 * i + i16;
      view.t[i] = r < a.R ? r / a.G : a.T;
    }
    __syncthreads();
    const uint16_t* ql = &q_rows[i16][8 * g];
    State<D, NT> st;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      // never -inf: keys of score -inf then weigh 0 also where nothing came before
      st.m[i] = -FLT_MAX;
      st.l[i] = 0.f;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) st.acc[i][n] = f32x4{};
    }

    // This wavefront's blocks, kWaves c + wv for chunks c of the piece: those with
    // drafts or the end of the sequence first, while the first whole one is under way.
    const int nblk = (ctx + kBlk - 1) / kBlk;
    const int end = kWaves * c1 < nblk ? kWaves * c1 : nblk;
    int bi = kWaves * c0 + wv;
    int edge = bi < end ? bi + (end - 1 - bi) / kWaves * kWaves : -1;  // the last one
    int whole = view.prefix / kBlk;  // blocks of which every row sees all
    whole = whole < end ? whole : end;
    Pages pg{a.table + static_cast<size_t>(b) * a.max_pages, kvh, -(1 << 30), 0};
    uint16_t* ta = tile_a[wv];
    uint16_t* tb = tile_b[wv];
    const bool any = bi < whole;
    if (edge >= whole) {
      load_tile<D, AUX>(tb, a, pg, edge, lane);
      pg.base = -(1 << 30);
    }
    if (any) load_tile<D, AUX>(ta, a, pg, bi, lane);
    wait_vmem_all();
    while (edge >= whole) {
      edge_block<D, NT>(tb, ql, a.scale, st, view, edge, lane);
      edge -= kWaves;
      if (edge < whole || edge < bi) break;
      Pages back{pg.row, kvh, -(1 << 30), 0};
      load_tile<D, AUX>(tb, a, back, edge, lane);
      wait_vmem_all();
    }
    // block bi has landed in ta; the next one goes into the other buffer
    if (any) {
      while (true) {
        const bool more_b = bi + kWaves < whole;
        if (more_b) load_tile<D, AUX>(tb, a, pg, bi + kWaves, lane);
        whole_block<D, NT>(ta, ql, a.scale, st, lane);
        if (!more_b) break;
        wait_vmem_all();
        bi += 2 * kWaves;
        const bool more_a = bi < whole;
        if (more_a) load_tile<D, AUX>(ta, a, pg, bi, lane);
        whole_block<D, NT>(tb, ql, a.scale, st, lane);
        if (!more_a) break;
        wait_vmem_all();
      }
    }

    // merge the wavefronts
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float lt = wave_sum_across_groups(st.l[i]);
      if (g == 0) {
        red_m[wv][16 * i + i16] = st.m[i];
        red_l[wv][16 * i + i16] = lt;
      }
    }
    const bool all = c0 == 0 && c1 == chunks;
    const size_t slot = 2 * static_cast<size_t>(w) + (piece > 0 ? 1 : 0);
    __syncthreads();  // the buffers are no longer read
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      typedef float Merge[kWaves][16][kPad];
      Merge& buf = *reinterpret_cast<Merge*>(i & 1 ? &tile_b : &tile_a);
#pragma unroll
      for (int n = 0; n < D / 16; ++n)
        *reinterpret_cast<f32x4*>(&buf[wv][i16][16 * n + 4 * g]) = st.acc[i][n];
      __syncthreads();
      for (int idx = threadIdx.x; idx < 16 * (D / 4); idx += kThreads) {
        const int row = idx / (D / 4);
        const int d = (idx - row * (D / 4)) * 4;
        const int r = 16 * i + row;
        float M = red_m[0][r];
#pragma unroll
        for (int k = 1; k < kWaves; ++k) M = fmaxf(M, red_m[k][r]);
        float L = 0.f;
        f32x4 o = {};
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
          const float wt = fast_exp2(red_m[k][r] - M);
          L += red_l[k][r] * wt;
          o += *reinterpret_cast<const f32x4*>(&buf[k][row][d]) * wt;
        }
        if (!all) {
          *reinterpret_cast<f32x4*>(a.part_o + (slot * kRows + r) * D + d) = o;
          if (d == 0) *reinterpret_cast<float2*>(a.part_ml + (slot * kRows + r) * 2) = {M, L};
          continue;
        }
        const int rr = tile * kRows + r;
        if (rr >= a.R) continue;
        const int t = rr / a.G;
        const int head = kvh * a.G + (rr - t * a.G);
        const size_t at = (static_cast<size_t>(b) * a.T + t) * a.NQ + head;
        const bool empty = t >= view.drafts || L == 0.f;
        const float inv = empty ? 0.f : 1.f / L;
        *reinterpret_cast<u32x2*>(a.out + at * D + d) =
            empty ? u32x2{0u, 0u}
                  : u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
        if (a.lse != nullptr && d == 0)
          a.lse[at] = empty ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
      }
    }
    if (a.W == 0) return;
    u0 = u1 < begin + chunks ? u1 : begin + chunks;
    if (u0 >= u1) return;
    begin += chunks;
    if (++tile == a.tiles) {
      tile = 0;
      if (++kvh == a.NKV) {
        kvh = 0;
        do {
          ++b;
        } while (b < a.B - 1 && uniform(seg[b + 1]) == uniform(seg[b]));
        chunks = uniform(seg[b + 1]) - uniform(seg[b]);
      }
    }
    __syncthreads();  // the next piece writes q_rows, red_m, red_l and the buffers
  }
}

// One wavefront per row: merges the pieces of its segment, where the split cut it;
// rows of sequences without tokens are written here.
template <int D>
__global__ __launch_bounds__(kThreads) void gqa_tree_reduce_kernel(TreeArgs a, int rows_per_tile) {
  constexpr int DPL = D / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const long long task = static_cast<long long>(blockIdx.x) * kWaves + uniform(threadIdx.x / kWave);
  if (task >= static_cast<long long>(a.B) * a.NKV * a.R) return;
  const int seg = static_cast<int>(task / a.R);
  const int rr = static_cast<int>(task - static_cast<long long>(seg) * a.R);
  const int b = seg / a.NKV;
  const int kvh = seg - b * a.NKV;
  const int tile = rr / rows_per_tile;
  const int r = rr - tile * rows_per_tile;
  // chunks before sequence b, of b, and of all
  int before = 0, chunks = 0, total = 0;
  for (int base = 0; base < a.B; base += kWave) {
    const int i = base + lane;
    const int n = i < a.B ? chunks_of(context_of(a, i)) : 0;
    const int x = wave_inclusive_scan(n, lane);
    if (b >= base && b < base + kWave) {
      before = total + __builtin_amdgcn_readlane(x - n, b - base);
      chunks = __builtin_amdgcn_readlane(n, b - base);
    }
    total += __builtin_amdgcn_readlane(x, kWave - 1);
  }
  const int t = rr / a.G;
  const int head = kvh * a.G + (rr - t * a.G);
  const size_t at = (static_cast<size_t>(b) * a.T + t) * a.NQ + head;
  uint16_t* o = a.out + at * D + lane * DPL;
  const int ctx = uniform(context_of(a, b));
  const bool dead = t >= uniform(drafts_of(a, b, ctx));
  const int per_b = a.NKV * a.tiles;
  long long first = 0, last = -1, S = 0, U = 1;
  int We = 1;
  if (chunks > 0) {
    U = static_cast<long long>(total) * per_b;
    We = static_cast<int>(U < a.W ? U : a.W);
    S = static_cast<long long>(before) * per_b +
        static_cast<long long>(kvh * a.tiles + tile) * chunks;
    first = group_of_unit(S, U, We);
    last = group_of_unit(S + chunks - 1, U, We);
    if (first == last) return;  // written by its workgroup
  }
  float M = -FLT_MAX, L = 0.f, acc[DPL] = {};
  for (long long w = first; w <= last; ++w) {
    // a segment that starts inside its first workgroup's range is that one's last piece
    const bool later = w == first && w * U / We < S;
    const size_t p = (2 * static_cast<size_t>(w) + (later ? 1 : 0)) * rows_per_tile + r;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + p * 2);
    const float mn = fmaxf(M, ml.x);
    const float f = fast_exp2(M - mn), wt = fast_exp2(ml.x - mn);
    M = mn;
    L = L * f + ml.y * wt;
    const float* po = a.part_o + p * D + lane * DPL;
#pragma unroll
    for (int d = 0; d < DPL; ++d) acc[d] = acc[d] * f + po[d] * wt;
  }
  const bool empty = dead || L == 0.f;
  const float inv = empty ? 0.f : 1.f / L;
#pragma unroll
  for (int d = 0; d < DPL; ++d) o[d] = empty ? static_cast<uint16_t>(0) : f2bf(acc[d] * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[at] = empty ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
}

// How a call is cut.
struct TreePlan {
  int nt;     // 16-row column tiles of a wavefront
  int tiles;  // row tiles of a (sequence, kv head)
  int W;      // workgroups of the split; 0: one per segment, no reduce launch
};

TreePlan plan_tree(int head_dim, int G, int T, int max_pages, int page_tokens) {
  const int R = T * G;
  TreePlan p;
  p.nt = R <= 16 ? 1 : (R <= 32 ? 2 : 4);
  p.tiles = (R + 16 * p.nt - 1) / (16 * p.nt);
  const long long cap = static_cast<long long>(max_pages) * page_tokens;
  p.W = cap <= 1024 ? 0 : device_cu_count() * (head_dim == 64 ? 2 : 1);  // all run at once
  return p;
}

bool tree_shape_ok(int batch, int num_q_heads, int num_kv_heads, int head_dim, int drafts,
                   int page_tokens, int max_pages) {
  return batch > 0 && batch <= kMaxBatch && num_kv_heads > 0 && num_q_heads > 0 &&
         num_q_heads % num_kv_heads == 0 && num_q_heads / num_kv_heads <= 16 &&
         (head_dim == 64 || head_dim == 128) && drafts > 0 && drafts <= kMaxDrafts &&
         is_pow2(page_tokens) && page_tokens >= 32 && page_tokens <= 4096 && max_pages > 0 &&
         static_cast<long long>(max_pages) * page_tokens < (1LL << 30) &&
         static_cast<long long>(batch) * num_q_heads * drafts < (1LL << 28);
}

size_t part_o_bytes(const TreePlan& p, int D) {
  return static_cast<size_t>(2) * p.W * 16 * p.nt * D * sizeof(float);
}

template <int D>
void launch_tree(const TreeArgs& a, const TreePlan& p, dim3 grid, hipStream_t stream) {
  // (a byte of K/V that one row tile alone reads is streamed past the caches)
  if (p.nt == 1)
    hipLaunchKernelGGL((gqa_tree_kernel<D, 1, 2>), grid, dim3(kThreads), 0, stream, a);
  else if (p.nt == 2)
    hipLaunchKernelGGL((gqa_tree_kernel<D, 2, 2>), grid, dim3(kThreads), 0, stream, a);
  else if (p.tiles == 1)
    hipLaunchKernelGGL((gqa_tree_kernel<D, 4, 2>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((gqa_tree_kernel<D, 4, 0>), grid, dim3(kThreads), 0, stream, a);
}

}  // namespace
}  // namespace voom

using namespace voom;

extern "C" size_t voom_paged_gqa_tree_workspace_bytes(int batch, int num_q_heads,
                                                      int num_kv_heads, int head_dim, int drafts,
                                                      int page_tokens, int max_pages) {
  if (!tree_shape_ok(batch, num_q_heads, num_kv_heads, head_dim, drafts, page_tokens, max_pages))
    return 0;
  const TreePlan p = plan_tree(head_dim, num_q_heads / num_kv_heads, drafts, max_pages, page_tokens);
  return part_o_bytes(p, head_dim) + static_cast<size_t>(2) * p.W * 16 * p.nt * 2 * sizeof(float);
}

extern "C" int voom_paged_gqa_tree(const void* q, const void* k_pool, const void* v_pool,
                                   const int32_t* block_table, const int32_t* ctx_lens,
                                   const int32_t* draft_lens, const uint8_t* mask,
                                   int mask_batch, void* out, float* lse, void* workspace,
                                   size_t ws_bytes, int batch, int num_q_heads, int num_kv_heads,
                                   int head_dim, int page_tokens, int max_pages, int num_slots,
                                   int drafts, float scale, hipStream_t stream) {
  const char* who = "paged_gqa_tree";
  VOOM_REQUIRE(q && k_pool && v_pool && block_table && ctx_lens && out,
               "%s: null pointer argument", who);
  VOOM_REQUIRE(num_slots > 0, "%s: empty page pool", who);
  VOOM_REQUIRE(
      tree_shape_ok(batch, num_q_heads, num_kv_heads, head_dim, drafts, page_tokens, max_pages),
      "%s: unsupported geometry (batch %d, heads %d/%d, head_dim %d, %d drafts, %d pages of %d)",
      who, batch, num_q_heads, num_kv_heads, head_dim, drafts, max_pages, page_tokens);
  VOOM_REQUIRE(mask == nullptr || mask_batch == 1 || mask_batch == batch,
               "%s: %d masks for %d sequences", who, mask_batch, batch);
  VOOM_REQUIRE(std::isfinite(scale), "%s: the scale must be finite", who);
  VOOM_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(k_pool) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v_pool) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 8 == 0,
               "%s: q and pools must be 16-byte aligned", who);
  const int G = num_q_heads / num_kv_heads;
  const TreePlan p = plan_tree(head_dim, G, drafts, max_pages, page_tokens);
  const size_t need = voom_paged_gqa_tree_workspace_bytes(
      batch, num_q_heads, num_kv_heads, head_dim, drafts, page_tokens, max_pages);
  VOOM_REQUIRE(need == 0 || (workspace != nullptr && ws_bytes >= need &&
                             reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               "%s: workspace %zu bytes < required %zu (16-byte aligned)", who, ws_bytes, need);
  TreeArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k_pool = static_cast<const uint16_t*>(k_pool);
  a.v_pool = static_cast<const uint16_t*>(v_pool);
  a.table = block_table;
  a.ctx = ctx_lens;
  a.lens = draft_lens;
  a.mask = mask;
  a.mask_stride = mask_batch == 1 ? 0 : static_cast<long long>(drafts) * drafts;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = need ? reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                              part_o_bytes(p, head_dim))
                   : nullptr;
  a.B = batch;
  a.NQ = num_q_heads;
  a.NKV = num_kv_heads;
  a.G = G;
  a.T = drafts;
  a.max_pages = max_pages;
  a.pt_shift = ilog2(page_tokens);
  a.num_slots = num_slots;
  a.R = drafts * G;
  a.tiles = p.tiles;
  a.W = p.W;
  const long long groups =
      p.W != 0 ? p.W : static_cast<long long>(batch) * num_kv_heads * p.tiles;
  a.per_xcd = static_cast<int>((groups + 7) / 8);
  a.scale = scale == 0.f ? 1.f : fabsf(scale) * 1.4426950408889634f;
  a.q_zero = scale == 0.f;
  a.q_flip = scale < 0.f ? 0x80008000u : 0u;
  const dim3 grid(static_cast<unsigned>(8 * a.per_xcd));
  if (head_dim == 128) launch_tree<128>(a, p, grid, stream);
  else launch_tree<64>(a, p, grid, stream);
  const int rc = VOOM_LAUNCH_CHECK("paged_gqa_tree: kernel launch");
  if (rc || p.W == 0) return rc;
  const long long rows = static_cast<long long>(batch) * num_kv_heads * a.R;
  const dim3 rgrid(static_cast<unsigned>((rows + kWaves - 1) / kWaves));
  if (head_dim == 128)
    hipLaunchKernelGGL(gqa_tree_reduce_kernel<128>, rgrid, dim3(kThreads), 0, stream, a,
                       16 * p.nt);
  else
    hipLaunchKernelGGL(gqa_tree_reduce_kernel<64>, rgrid, dim3(kThreads), 0, stream, a,
                       16 * p.nt);
  return VOOM_LAUNCH_CHECK("paged_gqa_tree: reduce launch");
}
