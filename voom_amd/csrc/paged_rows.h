// What the kernels share that hold a few rows of queries against a paged cache
// (gqa_tree.hip, gqa_chunk.hip): eight wavefronts, kRowWaves groups of 16 NT rows by
// kKeyWaves that take every other 32-token block, and K and V^T in the stages of a ring
// in LDS.  Per block, with the rows in the N dimension:
//   scores^T[token][row] = K . Q^T,  out^T[dim][row] += V^T . P^T   16x16x32 bf16
// Row 4g + r of score tile t holds token 8g + 4t + r, so that a lane's scores are
// the 8 consecutive tokens that its P^T operand needs.
#pragma once

#include "paged_ring.h"

#include <cfloat>
#include <cmath>

namespace voom {

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kKeyWaves = 2;  // wavefronts that share a group of rows
constexpr int kRowWaves = kWaves / kKeyWaves;
constexpr int kStages = 4;    // stages of the ring in LDS
constexpr int kStageElems = 2 * 64 * 128;  // of K and V^T
constexpr int stage_blocks(int D) { return kStageElems / (2 * kBlk * D); }
constexpr int stage_tokens(int D) { return stage_blocks(D) * kBlk; }

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
__device__ __forceinline__ void load_stage(uint16_t* stage, const uint16_t* k_pool,
                                           const uint16_t* v_pool, Pages& pg, int bi, int wv,
                                           int lane) {
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
    load_piece<AUX>((is_v ? v_pool : k_pool) + at * (kBlk * D), kBlk * D * 2,
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

// The reference maxima of a softmax are raised to those of the scores only where one is
// more than kSlack ahead: weights up to 2^kSlack lose nothing in bf16 and fp32, and
// after its first blocks a wavefront hardly ever rescales its sums.
constexpr float kSlack = 8.f;

// mx: the maxima of this lane's scores, log2 units.
template <int D, int NT>
__device__ __forceinline__ void raise_maxima(const float (&mx)[NT], State<D, NT>& st) {
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

template <int D, int NT>
__device__ __forceinline__ void products(const Operands<D>& o, const u32x4 (&p)[NT],
                                         State<D, NT>& st) {
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
      st.acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o.v[n]),
                                                             __builtin_bit_cast(bf16x8, p[i]),
                                                             st.acc[i][n], 0, 0, 0);
  }
}

// The same of a block where rows do not see some tokens, their weights P being 0:
// seen_of(i) gives the bits of this lane's 8 tokens that the row of tile i sees, `valid` of
// them lie before the context's end.  Tokens past the end are garbage and are cut out of
// V^T; where only some rows see a token, 0 times a NaN or an infinity is NaN: where V holds
// one it is taken out, and products of indicators (V is NaN, +inf, -inf; the row sees the
// token) say which sums it belongs to.  v_of(n) gives the V^T operand of dims 16 n ...
template <int D, int NT, class Read, class Seen>
__device__ __forceinline__ void masked_products(Read v_of, const u32x4 (&p)[NT],
                                                State<D, NT>& st, int valid, Seen seen_of) {
  uint32_t keep[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    keep[e] = (2 * e < valid ? 0xffffu : 0u) | (2 * e + 1 < valid ? 0xffff0000u : 0u);
  uint32_t odd = 0;  // not 0: V holds a NaN or an infinity
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    u32x4 v = v_of(n);
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
    const uint32_t seen = seen_of(i);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      ones[i][e] = ((seen >> 2 * e & 1) != 0 ? 0x3f80u : 0u) |
                   ((seen >> (2 * e + 1) & 1) != 0 ? 0x3f800000u : 0u);
  }
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    const u32x4 v = v_of(n);
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

}  // namespace voom
