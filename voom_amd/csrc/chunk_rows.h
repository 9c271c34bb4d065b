// What the kernels of attention over ragged chunks share (gqa_chunk.hip, gqa_chunk_token.hip,
// gqa_chunk_wide.hip): the call's arguments, which cached tokens a new one sees, and the
// score of a pair.
#pragma once

#include "common.h"

namespace voom {

constexpr int kMaxChunkBatch = 1024;  // sequences of a call

struct ChunkArgs {
  const uint16_t* q;       // packed [N, NQ, D], or [B, NQ, T, D]
  const uint16_t* k_pool;
  const uint16_t* v_pool;
  const int32_t* table;    // [B, max_pages]
  const int32_t* ctx;      // [B]
  const int32_t* starts;   // [B + 1] first rows of the sequences, packed; or null
  const int32_t* lens;     // [B] new tokens, not packed; or null: T each
  const float* slopes;     // [NQ], or null
  const int32_t* prefix;   // [B], or null
  uint16_t* out;           // [N, NQ, D], or [B, T, NQ, D]
  float* lse;              // the same without D, or null
  float* part_o;           // [pieces, rows, D]
  float* part_ml;          // [pieces, rows, 2]
  int B, NQ, NKV, G, T, N, max_pages, pt_shift, num_slots;
  int window;    // tokens, INT_MAX: no window
  float scale;   // softmax scale in log2 units
  float cap;     // score cap in log2 units, 0: none
  float cap_k;   // softmax scale / score cap
  int W;         // workgroups of the split, 0: one per segment
  int per_xcd;   // workgroups per XCD
};

__device__ __forceinline__ int clamped(int x, int most) {
  return x < 0 ? 0 : (x > most ? most : x);
}

__device__ __forceinline__ int context_of(const ChunkArgs& a, int b) {
  return clamped(a.ctx[b], a.max_pages << a.pt_shift);
}

// The new tokens of sequence b and its first row among the packed ones, both kept inside
// the arrays whatever starts holds.
__device__ __forceinline__ int new_of(const ChunkArgs& a, int b, int& base) {
  if (a.starts == nullptr) {
    base = 0;
    return clamped(a.lens != nullptr ? a.lens[b] : a.T, a.T);
  }
  base = clamped(a.starts[b], a.N);
  const int end = clamped(a.starts[b + 1], a.N);
  return end > base ? end - base : 0;
}

__device__ __forceinline__ int prefix_of(const ChunkArgs& a, int b, int ctx) {
  return a.prefix != nullptr ? clamped(a.prefix[b], ctx) : 0;
}

// Elements from one sequence's queries to the next token's and the next head's, and the
// row of out and lse of a (sequence, token, head).
__device__ __forceinline__ size_t query_at(const ChunkArgs& a, int b, int base, int t, int head) {
  return a.starts != nullptr ? static_cast<size_t>(base + t) * a.NQ + head
                             : (static_cast<size_t>(b) * a.NQ + head) * a.T + t;
}
__device__ __forceinline__ size_t out_at(const ChunkArgs& a, int b, int base, int t, int head) {
  return (a.starts != nullptr ? static_cast<size_t>(base + t) : static_cast<size_t>(b) * a.T + t) *
             a.NQ + head;
}

// The tokens [lo, hi) that token t of the newest n sees, and with them [0, pre) where that
// does not reach lo (else it is one range).  Both ends rise with t.
struct Sight {
  int at, lo, hi;
  __device__ __forceinline__ Sight(const ChunkArgs& a, int ctx, int n, int pre, int t) {
    at = ctx - n + t;  // (before the cache where there are more new tokens than cached ones)
    hi = at + 1 > 0 ? at + 1 : 0;
    lo = at < a.window ? 0 : at + 1 - a.window;
    if (pre > 0 && lo <= pre) {
      lo = 0;
      hi = hi > pre ? hi : pre;
    }
  }
};

// Bits of 8 consecutive tokens from pos on that lie in [lo, hi).
__device__ __forceinline__ uint32_t bits_in(int pos, int lo, int hi) {
  const int a = lo - pos, b = hi - pos;
  const uint32_t below = b >= 8 ? 0xffu : (b > 0 ? (1u << b) - 1 : 0u);
  const uint32_t before = a >= 8 ? 0xffu : (a > 0 ? (1u << a) - 1 : 0u);
  return below & ~before;
}

// tanh(x) / x for |x| <= kNear as a polynomial of x^2, off by 7.1e-8 at most, relative: found
// by Remez's exchange of the extrema of the relative error, which holds to 3.5e-8, its first
// term then rounded to 1, so that no small score is changed.
constexpr float kNear = 0.35f;
constexpr float kTanh[4] = {1.f, -0.33332422375679016f, 0.13295799493789673f,
                            -0.04895823076367378f};
__device__ __forceinline__ float tanh_ratio(float x2) {
  float p = __builtin_fmaf(kTanh[3], x2, kTanh[2]);
  p = __builtin_fmaf(p, x2, kTanh[1]);
  return __builtin_fmaf(p, x2, kTanh[0]);
}

// cap tanh(x) further out, where 1 - 2 / (e^2x + 1) loses nothing to cancellation.
__device__ __forceinline__ float capped_far(float x, float cap) {
  const float e = fast_exp2(x * 2.885390081777927f);
  return __builtin_fmaf(-2.f * cap, __builtin_amdgcn_rcpf(e + 1.f), cap);
}

// ---- the kernels of single tokens (gqa_chunk_token.hip) and short chunks ------------

// How a call with few rows is cut.
struct FewPlan {
  int rows;        // of a row tile
  long long segs;  // (sequence, kv head, row tile) segments at most
  int W;           // workers of the split; 0: one per segment, no reduce launch
};
FewPlan plan_token(int B, int NKV, int D, int G, int N, int T, long long tokens, int window);
int launch_token(const ChunkArgs& a, const FewPlan& p, int D, hipStream_t stream);

// ---- the kernel of long chunks (gqa_chunk_wide.hip) ------------------------------

// Its workspace, sized for any lengths that the call's rows allow.
struct WidePlan {
  int entries;     // (sequence, row tile) pairs at most
  int pieces;      // of a kv head at most, row tiles cut over keys
  int cuts;        // row tiles of a kv head that are cut, at most
  int slots;       // pieces of those
  int workers;     // workgroups that run at once
  size_t bytes;
};
WidePlan plan_wide(int B, int NKV, int D, int G, int N, int T, long long tokens);
int launch_wide(const ChunkArgs& a, const WidePlan& p, int D, void* workspace,
                hipStream_t stream);

}  // namespace voom
