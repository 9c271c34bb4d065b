// Head norms, rotary positions and the page write of new tokens, for gfx950.
//
// qkv [B * L, (nq + 2 nkv) * hd] holds the projections.  Every query and key head is
// normed, y = x / sqrt(mean x^2 + eps) * w (where a weight is given), its first rd
// dims are rotated by the angle of the token's position, and q is written to
// [B, nq, L, hd], k and v into their pages at the cache position start[b] + t:
//   half layout         dims (i, i + rd/2) form a pair
//   interleaved layout  dims (2 i, 2 i + 1) form a pair
//   (a, b) -> (a cos - b sin, b cos + a sin), cos and sin of row position, column i
// All of it in fp32, rounded to bf16 once.
//
// What bounds it: the projections read and q, k, v written once; one launch for a
// token's few heads.  Some workgroups take the query and key heads, 8 dims per lane; the
// others the value heads, a 32-token cache block each, which they transpose in LDS: V
// pages hold 64-byte rows of 32 tokens, and written element by element a prompt of
// 2,011 tokens (32/8 heads of 128) took 23 us where this takes 15.
#include "common.h"

namespace voom {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

struct QkArgs {
  const uint16_t* qkv;
  const uint16_t* q_weight;  // [hd], or null: no norm
  const uint16_t* k_weight;
  const float* cos_t;        // [P, rd / 2]
  const float* sin_t;
  const int32_t* positions;  // [B, L]
  uint16_t* q;
  uint16_t* k_pool;
  uint16_t* v_pool;
  const int32_t* table;      // [B, max_pages]
  const int32_t* start;      // [B]
  const int32_t* lens;       // [B], or null: L each
  float eps;
  int P, rd, interleaved, B, L, nq, nkv, hd, group_shift, pt_shift, max_pages, num_slots;
  int blocks;     // V blocks that the new tokens of a sequence can touch
  int qk_groups;  // workgroups of query and key heads, before those of V
};

__device__ __forceinline__ void unpack8(u32x4 x, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = __builtin_bit_cast(float, x[e] << 16);
    f[2 * e + 1] = __builtin_bit_cast(float, x[e] & 0xffff0000u);
  }
}

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = a[e];
    f[4 + e] = b[e];
  }
}

// Query and key heads: `group` lanes (a power of two, 8 dims each) per head of a token.
__device__ __forceinline__ void query_and_key_heads(const QkArgs& a) {
  const int heads = a.nq + a.nkv;
  const unsigned idx = blockIdx.x * kThreads + threadIdx.x;
  const int rh = static_cast<int>(idx >> a.group_shift);
  const int lane = static_cast<int>(idx & ((1u << a.group_shift) - 1));
  const int row = rh / heads;
  const int h = rh - row * heads;
  const bool in = row < a.B * a.L && 8 * lane < a.hd;
  const int b = in ? row / a.L : 0;
  const int t = in ? row - b * a.L : 0;
  const int d0 = in ? 8 * lane : 0;
  const uint16_t* src = a.qkv + (in ? static_cast<size_t>(row) * (heads + a.nkv) + h : 0) * a.hd;
  const u32x4 raw = *reinterpret_cast<const u32x4*>(src + d0);
  u32x4 o = raw;
  float x[8];
  unpack8(raw, x);
  const uint16_t* w = h < a.nq ? a.q_weight : a.k_weight;
  const int half = a.rd / 2;
  const bool turn = d0 < a.rd;
  // the dims that these turn with, half layout
  const int p0 = a.interleaved || !turn ? d0 : (d0 < half ? d0 + half : d0 - half);
  float y[8];
  unpack8(*reinterpret_cast<const u32x4*>(src + p0), y);
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = in ? __builtin_fmaf(x[e], x[e], ss) : 0.f;
    for (int k = 1; k < 1 << a.group_shift; k <<= 1) ss += __shfl_xor(ss, k);
    const float r = 1.f / sqrtf(ss / static_cast<float>(a.hd) + a.eps);
    float wx[8], wy[8];
    unpack8(*reinterpret_cast<const u32x4*>(w + d0), wx);
    unpack8(*reinterpret_cast<const u32x4*>(w + p0), wy);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = x[e] * r * wx[e];
      y[e] = y[e] * r * wy[e];
    }
  }
  if (turn) {
    int pos = a.positions[in ? row : 0];
    pos = pos < 0 ? 0 : (pos < a.P ? pos : a.P - 1);
    const size_t at = static_cast<size_t>(pos) * half;
    if (a.interleaved) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(a.cos_t + at + d0 / 2);
      const f32x4 s = *reinterpret_cast<const f32x4*>(a.sin_t + at + d0 / 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = x[2 * e], v = x[2 * e + 1];
        x[2 * e] = u * c[e] - v * s[e];
        x[2 * e + 1] = v * c[e] + u * s[e];
      }
    } else {
      const float sign = d0 < half ? -1.f : 1.f;
      float c[8], s[8];
      load8(a.cos_t + at + (d0 < half ? d0 : d0 - half), c);
      load8(a.sin_t + at + (d0 < half ? d0 : d0 - half), s);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * c[e] + sign * y[e] * s[e];
    }
  }
  if (w != nullptr || turn) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
  }
  if (!in) return;
  if (h < a.nq) {
    *reinterpret_cast<u32x4*>(a.q + ((static_cast<size_t>(b) * a.nq + h) * a.L + t) * a.hd + d0) =
        o;
    return;
  }
  if (a.lens != nullptr && t >= a.lens[b]) return;
  const long long pos = static_cast<long long>(a.start[b]) + t;
  if (a.start[b] < 0 || pos >= static_cast<long long>(a.max_pages) << a.pt_shift) return;
  const int off = static_cast<int>(pos) & ((1 << a.pt_shift) - 1);
  const int slot =
      a.table[static_cast<size_t>(b) * a.max_pages + (static_cast<int>(pos) >> a.pt_shift)];
  if (static_cast<unsigned>(slot) >= static_cast<unsigned>(a.num_slots)) return;
  const size_t at = ((static_cast<size_t>(slot) * a.nkv + (h - a.nq)) << a.pt_shift) + off;
  *reinterpret_cast<u32x4*>(a.k_pool + at * a.hd + d0) = o;
}

// One block of up to 32 consecutive cache positions of one (sequence, value head).
__device__ __forceinline__ void value_block(const QkArgs& a, int task) {
  __shared__ __attribute__((aligned(16))) uint16_t tile[32][kMaxDim + 8];
  const int vb = a.pt_shift < 5 ? a.pt_shift : 5;
  const int VB = 1 << vb;
  const int bh = task / a.blocks;
  const int j = task - bh * a.blocks;  // of the blocks that the sequence's tokens can touch
  const int b = bh / a.nkv;
  const int h = bh - b * a.nkv;
  int n = a.lens != nullptr ? uniform(a.lens[b]) : a.L;
  n = n < a.L ? n : a.L;
  const int start = uniform(a.start[b]);
  const int cap = a.max_pages << a.pt_shift;
  if (start < 0 || start >= cap) return;
  // tokens t0 .. t1 land in this block, at its columns c0 ..
  const int first = ((start >> vb) + j) << vb;  // cache position of the block
  const int t0 = first > start ? first - start : 0;
  int t1 = first + VB - start;
  t1 = t1 < n ? t1 : n;
  if (t0 >= t1 || first >= cap) return;
  const int c0 = start + t0 - first;
  const int slot = uniform(a.table[static_cast<size_t>(b) * a.max_pages + (first >> a.pt_shift)]);
  if (static_cast<unsigned>(slot) >= static_cast<unsigned>(a.num_slots)) return;
  const int chunks = a.hd / 8;
  const int heads = a.nq + 2 * a.nkv;
  for (int i = threadIdx.x; i < (t1 - t0) * chunks; i += kThreads) {
    const int t = i / chunks;
    const int c = i - t * chunks;
    *reinterpret_cast<u32x4*>(&tile[c0 + t][8 * c]) = *reinterpret_cast<const u32x4*>(
        a.qkv + ((static_cast<size_t>(b) * a.L + t0 + t) * heads + a.nq + a.nkv + h) * a.hd +
        8 * c);
  }
  __syncthreads();
  const size_t head_page = static_cast<size_t>(slot) * a.nkv + h;
  uint16_t* v = a.v_pool + (((head_page << (a.pt_shift - vb)) +
                             ((first & ((1 << a.pt_shift) - 1)) >> vb)) * a.hd << vb);
  if (t1 - t0 == 32) {  // whole rows of 32 tokens, 16 bytes per lane
    for (int i = threadIdx.x; i < a.hd * 4; i += kThreads) {
      const int d = i >> 2, g = i & 3;
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        o[e] = tile[8 * g + 2 * e][d] | static_cast<uint32_t>(tile[8 * g + 2 * e + 1][d]) << 16;
      *reinterpret_cast<u32x4*>(v + d * 32 + 8 * g) = o;
    }
    return;
  }
  for (int i = threadIdx.x; i < a.hd << vb; i += kThreads) {
    const int d = i >> vb, c = i & (VB - 1);
    if (c >= c0 && c < c0 + t1 - t0) v[i] = tile[c][d];
  }
}

__global__ __launch_bounds__(kThreads) void qk_norm_rope_append_kernel(QkArgs a) {
  const int task = static_cast<int>(blockIdx.x) - a.qk_groups;
  if (task < 0) query_and_key_heads(a);
  else value_block(a, task);
}

}  // namespace
}  // namespace voom

using namespace voom;

extern "C" int voom_qk_norm_rope_append(const void* qkv, const void* q_weight,
                                        const void* k_weight, float eps, const float* cos,
                                        const float* sin, int rope_rows, int rotary_dim,
                                        int interleaved, const int32_t* positions, void* q,
                                        void* k_pool, void* v_pool, const int32_t* block_table,
                                        const int32_t* start, const int32_t* new_lens, int batch,
                                        int new_tokens, int num_q_heads, int num_kv_heads,
                                        int head_dim, int page_tokens, int max_pages,
                                        int num_slots, hipStream_t stream) {
  const char* who = "qk_norm_rope_append";
  VOOM_REQUIRE(qkv && cos && sin && positions && q && k_pool && v_pool && block_table && start,
               "%s: null pointer argument", who);
  VOOM_REQUIRE(batch > 0 && new_tokens > 0 && num_q_heads > 0 && num_kv_heads > 0 &&
                   max_pages > 0 && num_slots > 0 && rope_rows > 0,
               "%s: bad geometry (batch %d, %d new tokens, heads %d/%d, %d rope rows)", who, batch,
               new_tokens, num_q_heads, num_kv_heads, rope_rows);
  VOOM_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim <= kMaxDim,
               "%s: head_dim %d must be a multiple of 16 up to 256", who, head_dim);
  VOOM_REQUIRE(rotary_dim > 0 && rotary_dim % 16 == 0 && rotary_dim <= head_dim,
               "%s: rotary_dim %d must be a multiple of 16 up to head_dim %d", who, rotary_dim,
               head_dim);
  VOOM_REQUIRE(is_pow2(page_tokens) && page_tokens <= 4096,
               "%s: page_tokens %d must be a power of two <= 4096", who, page_tokens);
  VOOM_REQUIRE(static_cast<long long>(max_pages) * page_tokens < (1LL << 30),
               "%s: block table of %d pages of %d tokens", who, max_pages, page_tokens);
  VOOM_REQUIRE(eps >= 0.f, "%s: eps must not be negative", who);
  for (const void* p : {qkv, q_weight, k_weight, static_cast<const void*>(cos),
                        static_cast<const void*>(sin), static_cast<const void*>(q),
                        static_cast<const void*>(k_pool), static_cast<const void*>(v_pool)})
    VOOM_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "%s: buffers must be 16-byte aligned",
                 who);
  QkArgs a;
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.q_weight = static_cast<const uint16_t*>(q_weight);
  a.k_weight = static_cast<const uint16_t*>(k_weight);
  a.cos_t = cos;
  a.sin_t = sin;
  a.positions = positions;
  a.q = static_cast<uint16_t*>(q);
  a.k_pool = static_cast<uint16_t*>(k_pool);
  a.v_pool = static_cast<uint16_t*>(v_pool);
  a.table = block_table;
  a.start = start;
  a.lens = new_lens;
  a.eps = eps;
  a.P = rope_rows;
  a.rd = rotary_dim;
  a.interleaved = interleaved;
  a.B = batch;
  a.L = new_tokens;
  a.nq = num_q_heads;
  a.nkv = num_kv_heads;
  a.hd = head_dim;
  a.group_shift = 0;
  while (8 << a.group_shift < head_dim) ++a.group_shift;
  a.pt_shift = ilog2(page_tokens);
  a.max_pages = max_pages;
  a.num_slots = num_slots;
  const int block_tokens = page_tokens < 32 ? page_tokens : 32;
  a.blocks = (new_tokens + block_tokens - 2) / block_tokens + 1;
  const long long lanes = static_cast<long long>(batch) * new_tokens *
                          (num_q_heads + static_cast<long long>(num_kv_heads)) << a.group_shift;
  const long long v_groups = static_cast<long long>(batch) * num_kv_heads * a.blocks;
  VOOM_REQUIRE(lanes < (1LL << 31) - kThreads && v_groups < (1LL << 30),
               "%s: too many heads of too many tokens in one call", who);
  a.qk_groups = static_cast<int>((lanes + kThreads - 1) / kThreads);
  const long long groups = a.qk_groups + v_groups;
  hipLaunchKernelGGL(qk_norm_rope_append_kernel, dim3(static_cast<unsigned>(groups)),
                     dim3(kThreads), 0, stream, a);
  return VOOM_LAUNCH_CHECK("qk_norm_rope_append: launch");
}
