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
// Work decomposition.  A workgroup takes 64 rows (128 where there are more) of a
// (sequence, kv head), so that up to 128 share every K/V byte.  A unit is a stage of
// 64 tokens (128 at D = 64) of one (sequence, kv head, row tile) segment; the units of
// all segments lie end to end, each after kLead that stand for what a segment costs
// besides, and workgroup w of W takes [w U/W, (w+1) U/W): all work as long whatever the
// context lengths (without kLead those with many short segments were the last: 17
// sequences of up to 2,247 tokens, 28 drafts, 64/8 heads, 113 us instead of 58).  A
// segment within one workgroup is written from there; of the others a workgroup holds at
// most two pieces, an end and a start, which gqa_tree_reduce_kernel merges.
//
// Eight wavefronts, two per SIMD, so that one's matrix work runs beside the other's
// exponentials: four groups of 16 NT rows, two wavefronts each, which take every
// other 32-token block.  K and V^T go straight into LDS (buffer_load ... lds, 1 KiB
// each) through a ring of four 32 KiB stages: three are under way while one is
// computed (a ring of two per wavefront drained it at every stage: 371 us at 16
// sequences of 1k-32k tokens, 16 drafts, 32/8 heads, where this takes 231; blocks
// in registers, as in the decode kernel, leave too few for 64 rows: 1,076).  Per block,
// with the rows in the N dimension:
//   scores^T[token][row] = K . Q^T,  out^T[dim][row] += V^T . P^T   16x16x32 bf16
// Row 4g + r of score tile t holds token 8g + 4t + r, so that a lane's scores are
// the 8 consecutive tokens that its P^T operand needs.
//
// P is rounded to bf16 for the matrix units; its sum, and with it the LSE, is kept
// of the unrounded fp32 weights (the roundings average out in the output, whose own
// rounding is as large as one of them).
#include "paged_ring.h"

#include <cfloat>
#include <cmath>

namespace voom {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeyWaves = 2;  // wavefronts that share a group of rows
constexpr int kRowWaves = kWaves / kKeyWaves;
constexpr int kStages = 4;    // stages of the ring in LDS
constexpr int kStageElems = 2 * 64 * 128;  // of K and V^T
constexpr int stage_blocks(int D) { return kStageElems / (2 * kBlk * D); }
constexpr int stage_tokens(int D) { return stage_blocks(D) * kBlk; }
constexpr int kLead = 8;      // units that a segment costs besides its chunks
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
  float* part_o;          // [2 W, rows, D]
  float* part_ml;         // [2 W, rows, 2]
  long long mask_stride;  // elements from one sequence's mask to the next
  int B, NQ, NKV, G, T, max_pages, pt_shift, num_slots;
  int R;         // rows of a (sequence, kv head): T * G, (draft, head), head fastest
  int rows;      // rows of a tile
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

// Units of a context.
template <int D>
__device__ __forceinline__ int chunks_of(int ctx) {
  return (ctx + stage_tokens(D) - 1) / stage_tokens(D);
}

// Units of a sequence: for every kv head and row tile that holds a draft its chunks, after
// kLead units that stand for what a segment costs besides (queries, the first loads of an
// empty ring, drafts and masks, the merge).
template <int D>
struct Units {
  int chunks, tiles;
  __device__ __forceinline__ int all(const TreeArgs& a) const {
    return chunks == 0 ? 0 : (chunks + kLead) * tiles * a.NKV;
  }
  __device__ __forceinline__ Units(const TreeArgs& a, int b) {
    const int ctx = context_of(a, b);
    chunks = chunks_of<D>(ctx);
    const int t = (drafts_of(a, b, ctx) * a.G + a.rows - 1) >> (a.rows == 128 ? 7 : 6);
    tiles = t < 1 ? 1 : t;
  }
};

// The units of up to 64 sequences from `base` on, one per lane, and their inclusive sum.
template <int D>
__device__ __forceinline__ Units<D> scan_units(const TreeArgs& a, int base, int lane, int& x) {
  const bool in = base + lane < a.B;
  const Units<D> u(a, in ? base + lane : 0);
  x = wave_inclusive_scan(in ? u.all(a) : 0, lane);
  return u;
}

// Chunk c (16 bytes) of K row r sits at c ^ k_swizzle(r) of its row, chunk c of V^T row
// d at c ^ v_swizzle(d >> 2): the rows of an operand read then spread over all banks,
// whether 16 consecutive lanes are served together or lanes 0-3, 12-15, 20-27 (as d >> 2
// itself does not: two cycles of conflicts per read).
template <int D>
__device__ __forceinline__ int k_swizzle(int r) {
  return D == 128 ? (r & 3) | ((r >> 3) & 3) << 2 : ((r >> 1) & 1) | ((r >> 3) & 3) << 1;
}

__device__ __forceinline__ int v_swizzle(int h) {  // 0, 2, 3, 1
  h &= 3;
  return ((h ^ h >> 1) & 1) << 1 | h >> 1;
}

// A block of a stage in LDS: K [32][D], then V^T [D][32].
constexpr int block_elems(int D) { return 2 * kBlk * D; }

// Starts this wavefront's loads (of 1 KiB) of the stage whose first block is bi; blocks
// past the context repeat its last one, and are not used.
template <int D, int AUX>
__device__ __forceinline__ void load_stage(uint16_t* stage, const TreeArgs& a, Pages& pg, int bi,
                                           int wv, int lane) {
  constexpr int kBlocks = stage_blocks(D);
  constexpr int kPieces = kBlk * D / 512;  // of K, and of V^T, of a block
  constexpr int kCpr = D / 8;              // 16-byte chunks of a K row
  pg.hold(bi, kBlocks, lane);
#pragma unroll
  for (int i = 0; i < 2 * kBlocks * kPieces / kWaves; ++i) {
    // piece p = wv + 8 i: block p / (2 kPieces), first its K and then its V^T
    const int p = wv + kWaves * i;
    const int in_blk = p % (2 * kPieces);
    const size_t at = pg.block(bi + p / (2 * kPieces));
    const bool is_v = in_blk >= kPieces;
    const int sub = in_blk % kPieces;
    const int krow = sub * (kWave / kCpr) + lane / kCpr;
    const int ksrc = krow * (D * 2) + 16 * ((lane % kCpr) ^ k_swizzle<D>(krow));
    const int vsrc =
        sub * 1024 + (lane >> 2) * (kBlk * 2) + 16 * ((lane & 3) ^ v_swizzle(lane >> 4));
    load_piece<AUX>((is_v ? a.v_pool : a.k_pool) + at * (kBlk * D), kBlk * D * 2,
                    is_v ? vsrc : ksrc, stage + p * 512);
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
                                         8 * (g ^ v_swizzle(i16 >> 2)));
}

// A block's K and V^T operands.
template <int D>
struct Operands {
  u32x4 k[D / 32][2];
  u32x4 v[D / 16];
};

template <int D>
__device__ __forceinline__ void read_keys(Operands<D>& o, const uint16_t* tile, int lane) {
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
#pragma unroll
    for (int t = 0; t < 2; ++t) o.k[s][t] = read_k<D>(tile, t, s, lane);
  }
}

template <int D>
__device__ __forceinline__ void read_block(Operands<D>& o, const uint16_t* tile, int lane) {
  read_keys<D>(o, tile, lane);
#pragma unroll
  for (int n = 0; n < D / 16; ++n) o.v[n] = read_v<D>(tile, n, lane);
  __builtin_amdgcn_sched_barrier(0);  // all of them on their way before the first is waited for
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
  // Bit e: the row of tile i sees token pos + e, e < 8.  Bytes beside the row are read and
  // not used; outside the sequence's mask the buffer gives 0.
  __device__ __forceinline__ uint32_t seen(int i, int pos) const {
    const int j = pos - prefix;
    uint32_t bits = 0;
    if (mask != nullptr) {
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(mask), static_cast<short>(0), T * T, 0x00020000);
      uint8_t m[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        m[e] = __builtin_amdgcn_raw_buffer_load_b8(r, t[i] * T + j + e, 0, 0);
#pragma unroll
      for (int e = 0; e < 8; ++e) bits |= (m[e] != 0 ? 1u : 0u) << e;
    } else {
      const int n = t[i] - j + 1;  // tokens up to the draft's own
      bits = n >= 8 ? 0xffu : (n > 0 ? (1u << n) - 1 : 0u);
    }
    const int d = drafts - j;  // tokens up to the context's end
    bits &= d >= 8 ? 0xffu : (d > 0 ? (1u << d) - 1 : 0u);
    const int before = -j;     // tokens before the drafts
    bits |= before >= 8 ? 0xffu : (before > 0 ? (1u << before) - 1 : 0u);
    return t[i] < drafts ? bits : 0u;
  }
};

template <int D, int NT>
__device__ __forceinline__ void scores_of(const Operands<D>& o, const u32x4 (&qop)[NT][D / 32],
                                          f32x4 (&sc)[NT][2]) {
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    sc[i][0] = f32x4{};
    sc[i][1] = f32x4{};
  }
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        sc[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o.k[s][t]),
                                                           __builtin_bit_cast(bf16x8, qop[i][s]),
                                                           sc[i][t], 0, 0, 0);
    }
  }
}

// Forms P.  The reference maxima are raised to those of the scores only where one is
// more than kSlack ahead: weights up to 2^kSlack lose nothing in bf16 and fp32, and
// after its first blocks a wavefront hardly ever rescales its sums.
constexpr float kSlack = 8.f;

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
    up |= mx[i] > st.m[i] + kSlack;
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
__device__ __forceinline__ void whole_block(const Operands<D>& o,
                                            const u32x4 (&qop)[NT][D / 32], float scale,
                                            State<D, NT>& st) {
  f32x4 sc[NT][2];
  u32x4 p[NT];
  scores_of<D, NT>(o, qop, sc);
  weights_of<D, NT>(sc, scale, st, p);
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
      st.acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o.v[n]),
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
__device__ __forceinline__ void edge_block(const uint16_t* tile,
                                           const u32x4 (&qop)[NT][D / 32], float scale,
                                           State<D, NT>& st, const View<NT>& view, int bi,
                                           int lane) {
  const int g = lane >> 4;
  f32x4 sc[NT][2];
  u32x4 p[NT];
  {
    Operands<D> o;
    read_keys<D>(o, tile, lane);
    scores_of<D, NT>(o, qop, sc);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const uint32_t seen = view.seen(i, bi * kBlk + 8 * g);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sc[i][e >> 2][e & 3] = (seen >> e & 1) != 0 ? sc[i][e >> 2][e & 3] : -INFINITY;
    __builtin_amdgcn_sched_barrier(0);
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
    const uint32_t seen = view.seen(i, bi * kBlk + 8 * g);
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

template <int D, int NT, int AUX>
__global__ __launch_bounds__(kThreads, 2) void gqa_tree_kernel(TreeArgs a) {
  constexpr int kRows = 16 * NT * kRowWaves;
  constexpr int kBlocks = stage_blocks(D);
  constexpr int kLoads = 2 * kBlocks * (kBlk * D / 512) / kWaves;  // a wavefront's, of a stage
  constexpr int kPad = D + 4;  // floats of a row in LDS: 16 rows start in 16 bank groups
  // The ring.  Distinct objects, so that reads of one provably miss the pending
  // direct-to-LDS loads of the others; the merge uses them when the loop is done.
  __shared__ __attribute__((aligned(1024))) uint16_t stage_0[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_1[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_2[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_3[kStageElems];
  static_assert(kLoads == 4, "the waits below count the loads of a stage");
  static_assert(sizeof(float) * NT * 16 * kPad <= sizeof(stage_0), "a merge buffer fits a stage");

  const int lane = threadIdx.x & (kWave - 1);
  const int wv = uniform(threadIdx.x / kWave) & (kWaves - 1);
  const int kw = wv % kKeyWaves;
  const int rw = wv / kKeyWaves;
  const int i16 = lane & 15;
  const int g = lane >> 4;
  // Consecutive workgroups of one XCD take consecutive units, so that the row tiles
  // that read the same keys share an L2.
  const int bid = static_cast<int>(blockIdx.x);
  const int w = (bid & 7) * a.per_xcd + (bid >> 3);

  int b = 0, kvh, tile, c0, c1, chunks = 0, tiles = a.tiles;
  int u0 = 0, u1 = 0, begin = 0;  // the workgroup's units, and the segment's first one
  if (a.W == 0) {
    if (w >= a.B * a.NKV * tiles) return;
    b = w / (a.NKV * tiles);
    const int s = w - b * (a.NKV * tiles);
    kvh = s / tiles;
    tile = s - kvh * tiles;
    const Units<D> units(a, b);
    chunks = tile < uniform(units.tiles) ? uniform(units.chunks) : 0;
  } else {
    int x0;  // (every wavefront for itself: no barrier)
    const Units<D> first = scan_units<D>(a, 0, lane, x0);
    int U = __builtin_amdgcn_readlane(x0, kWave - 1);
    for (int base = kWave; base < a.B; base += kWave) {
      int x;
      scan_units<D>(a, base, lane, x);
      U += __builtin_amdgcn_readlane(x, kWave - 1);
    }
    const Split split(U, a.W);
    if (w >= split.We || U == 0) return;
    u0 = split.begin(w);
    u1 = split.begin(w + 1);
    for (int base = 0;; base += kWave) {  // the sequence that holds unit u0
      int x = x0;
      Units<D> units = first;
      if (base != 0) units = scan_units<D>(a, base, lane, x);
      const int here = __builtin_amdgcn_readlane(x, kWave - 1);
      if (u0 < begin + here) {
        const int k = __popcll(__builtin_amdgcn_ballot_w64(begin + x <= u0));
        b = base + k;
        chunks = __builtin_amdgcn_readlane(units.chunks, k);
        tiles = __builtin_amdgcn_readlane(units.tiles, k);
        begin += __builtin_amdgcn_readlane(x, k) - (chunks + kLead) * tiles * a.NKV;
        break;
      }
      begin += here;
    }
    const int s = (u0 - begin) / (chunks + kLead);
    kvh = s / tiles;
    tile = s - kvh * tiles;
    begin += s * (chunks + kLead);
  }
  while (true) {
    if (a.W == 0) {
      c0 = 0;
      c1 = chunks;
    } else {
      const int first = begin + kLead;  // the segment's first chunk
      if (u1 <= first) return;
      c0 = u0 > first ? u0 - first : 0;
      c1 = (u1 < first + chunks ? u1 : first + chunks) - first;
    }
    const int ctx = uniform(context_of(a, b));
    View<NT> view;
    view.ctx = ctx;
    view.drafts = uniform(drafts_of(a, b, ctx));
    view.prefix = ctx - view.drafts;
    view.mask = a.mask != nullptr ? a.mask + a.mask_stride * b : nullptr;
    view.T = a.T;
    // Q^T operands of this wavefront's rows
    u32x4 qop[NT][D / 32];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int r = tile * kRows + rw * (16 * NT) + 16 * i + i16;
      const int t = (r < a.R ? r : 0) / a.G;
      view.t[i] = r < a.R ? t : a.T;
      const int head = kvh * a.G + (r < a.R ? r - t * a.G : 0);
      const uint16_t* qr = a.q + ((static_cast<size_t>(b) * a.NQ + head) * a.T + t) * D + 8 * g;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        qop[i][s] = *reinterpret_cast<const u32x4*>(qr + 32 * s);
#pragma unroll
        for (int e = 0; e < 4; ++e) qop[i][s][e] ^= a.q_flip;
      }
    }
    if (a.q_zero) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
#pragma unroll
          for (int e = 0; e < 4; ++e) qop[i][s][e] = nan_bf16(qop[i][s][e]);
        }
      }
    }
    State<D, NT> st;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      // never -inf: keys of score -inf then weigh 0 also where nothing came before
      st.m[i] = -FLT_MAX;
      st.l[i] = 0.f;
#pragma unroll
      for (int n = 0; n < D / 16; ++n) st.acc[i][n] = f32x4{};
    }

    // Stages c0 .. c1.  Those with drafts or the end of the context come first, one at a
    // time through stage_3 while the first of the others are under way; of the others
    // every row sees all, and stage t of them is in t % 4.
    const int last_blk = (ctx - 1) / kBlk;
    Pages pg(a.table + static_cast<size_t>(b) * a.max_pages, a.max_pages, a.num_slots, a.NKV, kvh,
             a.pt_shift - 5, last_blk);
    int whole = view.prefix / stage_tokens(D);
    whole = whole < c1 ? whole : c1;
    // (else this wavefront only loads)
    const bool rows_here = tile * kRows + rw * (16 * NT) < view.drafts * a.G;
    int t = c0;
    auto load = [&](int at, uint16_t* stage) {
      load_stage<D, AUX>(stage, a, pg, at * kBlocks, wv, lane);
    };
    if (t < whole) load(t, stage_0);
    if (t + 1 < whole) load(t + 1, stage_1);
    if (t + 2 < whole) load(t + 2, stage_2);
#pragma unroll 1
    for (int e = whole > c0 ? whole : c0; e < c1; ++e) {
      load(e, stage_3);
      wait_vmem_all();
      lds_barrier();
      if (rows_here) {
#pragma unroll 1
        for (int j = kw; j < kBlocks && e * kBlocks + j <= last_blk; j += kKeyWaves)
          edge_block<D, NT>(stage_3 + j * block_elems(D), qop, a.scale, st, view, e * kBlocks + j,
                            lane);
      }
      lds_barrier();  // stage_3 is loaded again
    }
    auto step = [&](const uint16_t* cur, uint16_t* free) {
      // Stage t has landed for every wavefront, and stage t - 1 is no longer read.  gfx9
      // encoding: vmcnt of the loads of stages t + 1 and t + 2, expcnt 7, lgkmcnt 15.
      if (t + 2 < whole) __builtin_amdgcn_s_waitcnt(0x0F78);
      else if (t + 1 < whole) __builtin_amdgcn_s_waitcnt(0x0F74);
      else __builtin_amdgcn_s_waitcnt(0x0F70);
      lds_barrier();
      Operands<D> o;  // (the next loads are prepared while the first operands come)
      read_block<D>(o, cur + kw * block_elems(D), lane);
      if (t + 3 < whole) load(t + 3, free);
#pragma unroll
      for (int j = 0; j < kBlocks / kKeyWaves && rows_here; ++j) {
        if (j != 0) read_block<D>(o, cur + (kKeyWaves * j + kw) * block_elems(D), lane);
        whole_block<D, NT>(o, qop, a.scale, st);
      }
      return ++t < whole;
    };
    if (t < whole) {
      while (step(stage_0, stage_3) && step(stage_1, stage_0) && step(stage_2, stage_1) &&
             step(stage_3, stage_2)) {
      }
    }
    wait_vmem_all();
    lds_barrier();  // the ring is no longer read or written

    // Merge the two wavefronts of each group of rows: one leaves its state in LDS, the
    // other adds its own and writes.
    const bool all = c0 == 0 && c1 == chunks;
    const size_t slot = 2 * static_cast<size_t>(w) + (c0 == 0 ? 1 : 0);
    uint16_t* const merge = rw < 2 ? (rw == 0 ? stage_0 : stage_1) : (rw == 2 ? stage_2 : stage_3);
    float lt[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) lt[i] = wave_sum_across_groups(st.l[i]);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float* const buf = reinterpret_cast<float*>(merge) + i * 16 * kPad;
      if (kw == 1) {
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
          *reinterpret_cast<f32x4*>(buf + i16 * kPad + 16 * n + 4 * g) = st.acc[i][n];
        if (g == 0) {
          buf[i16 * kPad + D] = st.m[i];
          buf[i16 * kPad + D + 1] = lt[i];
        }
      }
    }
    __syncthreads();
    if (kw == 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const float* const buf = reinterpret_cast<const float*>(merge) + (i * 16 + i16) * kPad;
        const float m1 = buf[D];
        const float M = fmaxf(st.m[i], m1);
        const float f0 = fast_exp2(st.m[i] - M), f1 = fast_exp2(m1 - M);
        const float L = lt[i] * f0 + buf[D + 1] * f1;
        const int r = rw * (16 * NT) + 16 * i + i16;
        const int rr = tile * kRows + r;
        const int t_row = view.t[i];
        const bool empty = t_row >= view.drafts || L == 0.f;
        const float inv = 1.f / L;
        const int head = kvh * a.G + (rr - t_row * a.G);
        const size_t at = (static_cast<size_t>(b) * a.T + t_row) * a.NQ + head;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          const f32x4 o =
              st.acc[i][n] * f0 + *reinterpret_cast<const f32x4*>(buf + 16 * n + 4 * g) * f1;
          if (!all) {  // (rows past R too: they are in the workspace)
            *reinterpret_cast<f32x4*>(a.part_o + (slot * kRows + r) * D + 16 * n + 4 * g) = o;
          } else if (rr < a.R) {
            *reinterpret_cast<u32x2*>(a.out + at * D + 16 * n + 4 * g) =
                empty ? u32x2{0u, 0u}
                      : u32x2{pack_bf16x2(o[0] * inv, o[1] * inv),
                              pack_bf16x2(o[2] * inv, o[3] * inv)};
          }
        }
        if (g == 0 && !all)
          *reinterpret_cast<float2*>(a.part_ml + (slot * kRows + r) * 2) = {M, L};
        if (g == 0 && all && rr < a.R && a.lse != nullptr)
          a.lse[at] = empty ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
      }
    }
    if (a.W == 0) return;
    begin += kLead + chunks;
    u0 = u1 < begin ? u1 : begin;
    if (u0 >= u1) return;
    if (++tile == tiles) {
      tile = 0;
      if (++kvh == a.NKV) {
        kvh = 0;
        do {
          const Units<D> units(a, ++b);
          chunks = uniform(units.chunks);
          tiles = uniform(units.tiles);
        } while (b < a.B - 1 && chunks == 0);
      }
    }
    __syncthreads();  // the next piece writes the ring
  }
}

constexpr int kReduceWaves = 4;

// One wavefront per row: merges the pieces of its segment, where the split cut it; rows
// past their sequence's drafts become 0 here, in whichever tile (their wavefronts end before
// the search for the pieces: 17 sequences of up to 2,247 tokens, 28 drafts of 64/8 heads, 59
// us instead of 62).
template <int D>
__global__ __launch_bounds__(kReduceWaves * kWave) void gqa_tree_reduce_kernel(TreeArgs a) {
  // A wavefront holds the row of kTogether pieces at a time, 4 dims per lane.
  constexpr int kLanes = D / 4;
  constexpr int kTogether = kWave / kLanes;
  constexpr int kAhead = 8;  // loads in flight
  const int lane = threadIdx.x & (kWave - 1);
  const int b = static_cast<int>(blockIdx.z);
  const int kvh = static_cast<int>(blockIdx.y);
  const int rr = static_cast<int>(blockIdx.x) * kReduceWaves + uniform(threadIdx.x / kWave);
  if (rr >= a.R) return;
  const int tile = a.rows == 128 ? rr >> 7 : rr >> 6;
  const int r = rr & (a.rows - 1);
  const int t = rr / a.G;
  const int head = kvh * a.G + (rr - t * a.G);
  const size_t at = (static_cast<size_t>(b) * a.T + t) * a.NQ + head;
  const int sub = lane / kLanes;
  const int dim = lane % kLanes * 4;
  int first = 0, last = -1;
  const int ctx = uniform(context_of(a, b));
  if (t < uniform(drafts_of(a, b, ctx))) {  // (else 0, whoever else writes it)
    // units before sequence b, and of all; chunks and row tiles of b
    int before = 0, chunks = 0, tiles = 1, U = 0;
    for (int base = 0; base < a.B; base += kWave) {
      int x;
      const Units<D> units = scan_units<D>(a, base, lane, x);
      if (b >= base && b < base + kWave) {
        chunks = __builtin_amdgcn_readlane(units.chunks, b - base);
        tiles = __builtin_amdgcn_readlane(units.tiles, b - base);
        before = U + __builtin_amdgcn_readlane(x, b - base) - (chunks + kLead) * tiles * a.NKV;
      }
      U += __builtin_amdgcn_readlane(x, kWave - 1);
    }
    const Split split(U, a.W);
    const int S = before + (kvh * tiles + tile) * (chunks + kLead) + kLead;
    first = split.group(S);
    last = split.group(S + chunks - 1);
    if (first == last) return;  // written by its workgroup
  }
  // Up to 64 pieces at a time, one per lane for their maxima and sums.  A workgroup leaves
  // the piece that starts a segment, its last one, in its second slot.
  float M = -FLT_MAX, L = 0.f;
  f32x4 acc = {};
  for (int w0 = first; w0 <= last; w0 += kWave) {
    const int n = last - w0 + 1 < kWave ? last - w0 + 1 : kWave;
    const size_t p0 = 2 * static_cast<size_t>(w0) * a.rows + r;
    const int odd = w0 == first ? a.rows : 0;  // of the first one
    auto row_at = [&](int k) {
      k = k < n ? k : n - 1;
      return p0 + 2 * static_cast<size_t>(k) * a.rows + (k == 0 ? odd : 0);
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
    const float mn = fmaxf(M, wave_max_uniform(lane < n ? ml.x : -FLT_MAX));
    const float wt = lane < n ? fast_exp2(ml.x - mn) : 0.f;
    const float f = fast_exp2(M - mn);
    M = mn;
    L = L * f + wave_sum_uniform(lane < n ? ml.y * wt : 0.f);
    acc *= f;
    for (int k0 = 0; k0 < n; k0 += kAhead * kTogether) {
      if (k0 != 0) read(k0);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u * kTogether + sub;
        const float ws = __shfl(wt, k & (kWave - 1));
        if (k < n) acc += v[u] * ws;  // (0 times the infinity of a piece read again is NaN)
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

// How a call is cut.
struct TreePlan {
  int nt;     // 16-row tiles of a wavefront
  int rows;   // rows of a workgroup
  int tiles;  // row tiles of a (sequence, kv head)
  int W;      // workgroups of the split; 0: one per segment, no reduce launch
};

constexpr int kShort = 8, kLong = 64;  // stages of a segment that is not cut

TreePlan plan_tree(int B, int NKV, int D, int G, int T, int max_pages, int page_tokens) {
  const int R = T * G;
  TreePlan p;
  p.nt = R <= 64 ? 1 : 2;
  p.rows = 16 * p.nt * kRowWaves;
  p.tiles = (R + p.rows - 1) / p.rows;
  const long long stages = (static_cast<long long>(max_pages) * page_tokens + 64 * 128 / D - 1) /
                           (64 * 128 / D);
  const long long segs = static_cast<long long>(B) * NKV * p.tiles;
  // All workgroups of a split run at once.  Without one a workgroup walks a segment, which
  // saves the merges and the reduce launch: where the segments are short (8 heads, 8 stages:
  // 12.0 us so, 12.7 split; 12 stages: 13.4 and 12.4; 16: 20 and 14), the longer the better
  // they fill the card (192 of up to 9 stages: 14 and 21; 256 of up to 63: 61 and 72; 184
  // of up to 64: 76 and 51).
  const int cus = device_cu_count();
  const long long full = (segs + cus - 1) / cus * cus;
  const int most = 16 * segs >= 15 * full ? kLong : (2 * segs >= full ? 2 * kShort : kShort);
  p.W = stages <= most ? 0 : cus;
  return p;
}

bool tree_shape_ok(int batch, int num_q_heads, int num_kv_heads, int head_dim, int drafts,
                   int page_tokens, int max_pages) {
  return batch > 0 && batch <= kMaxBatch && num_kv_heads > 0 && num_kv_heads <= 65535 &&
         num_q_heads > 0 && num_q_heads % num_kv_heads == 0 &&
         num_q_heads / num_kv_heads <= 16 &&
         (head_dim == 64 || head_dim == 128) && drafts > 0 && drafts <= kMaxDrafts &&
         is_pow2(page_tokens) && page_tokens >= 32 && page_tokens <= 4096 && max_pages > 0 &&
         static_cast<long long>(max_pages) * page_tokens < (1LL << 30) &&
         static_cast<long long>(batch) * num_q_heads * drafts < (1LL << 28);
}

size_t part_o_bytes(const TreePlan& p, int D) {
  return static_cast<size_t>(2) * p.W * p.rows * D * sizeof(float);
}

template <int D>
void launch_tree(const TreeArgs& a, const TreePlan& p, dim3 grid, hipStream_t stream) {
  // (a byte of K/V that one row tile alone reads is streamed past the caches)
  if (p.nt == 1)
    hipLaunchKernelGGL((gqa_tree_kernel<D, 1, 2>), grid, dim3(kThreads), 0, stream, a);
  else if (p.tiles == 1)
    hipLaunchKernelGGL((gqa_tree_kernel<D, 2, 2>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((gqa_tree_kernel<D, 2, 0>), grid, dim3(kThreads), 0, stream, a);
}

}  // namespace
}  // namespace voom

using namespace voom;

extern "C" size_t voom_paged_gqa_tree_workspace_bytes(int batch, int num_q_heads,
                                                      int num_kv_heads, int head_dim, int drafts,
                                                      int page_tokens, int max_pages) {
  if (!tree_shape_ok(batch, num_q_heads, num_kv_heads, head_dim, drafts, page_tokens, max_pages))
    return 0;
  const TreePlan p = plan_tree(batch, num_kv_heads, head_dim, num_q_heads / num_kv_heads, drafts,
                               max_pages, page_tokens);
  return part_o_bytes(p, head_dim) + static_cast<size_t>(2) * p.W * p.rows * 2 * sizeof(float);
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
  const TreePlan p = plan_tree(batch, num_kv_heads, head_dim, G, drafts, max_pages, page_tokens);
  const long long stages = (static_cast<long long>(max_pages) * page_tokens + 63) / 64;
  VOOM_REQUIRE((stages + kLead) * batch * num_kv_heads * p.tiles < (1LL << 31),
               "%s: %d pages of %d tokens for %d sequences are too many", who, max_pages,
               page_tokens, batch);
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
  a.rows = p.rows;
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
  const dim3 rgrid(static_cast<unsigned>((a.R + kReduceWaves - 1) / kReduceWaves),
                   static_cast<unsigned>(num_kv_heads), static_cast<unsigned>(batch));
  if (head_dim == 128)
    hipLaunchKernelGGL(gqa_tree_reduce_kernel<128>, rgrid, dim3(kReduceWaves * kWave), 0, stream,
                       a);
  else
    hipLaunchKernelGGL(gqa_tree_reduce_kernel<64>, rgrid, dim3(kReduceWaves * kWave), 0, stream,
                       a);
  return VOOM_LAUNCH_CHECK("paged_gqa_tree: reduce launch");
}
