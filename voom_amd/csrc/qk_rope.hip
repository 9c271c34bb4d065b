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
// token's few heads.
#include "common.h"

namespace voom {
namespace {

constexpr int kThreads = 256;

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
  int P, rd, interleaved, B, L, nq, nkv, hd, group, pt_shift, max_pages, num_slots;
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

// `group` lanes (a power of two, 8 dims each) per head of a token.
__global__ __launch_bounds__(kThreads) void qk_norm_rope_append_kernel(QkArgs a) {
  const int heads = a.nq + 2 * a.nkv;
  const long long idx = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const long long rh = idx / a.group;
  const int lane = static_cast<int>(idx - rh * a.group);
  const long long row = rh / heads;
  const int h = static_cast<int>(rh - row * heads);
  const bool in = row < static_cast<long long>(a.B) * a.L && 8 * lane < a.hd;
  const int b = in ? static_cast<int>(row / a.L) : 0;
  const int t = in ? static_cast<int>(row - static_cast<long long>(b) * a.L) : 0;
  const int d0 = in ? 8 * lane : 0;
  const uint16_t* src = a.qkv + (in ? rh : 0) * a.hd;
  const u32x4 raw = *reinterpret_cast<const u32x4*>(src + d0);
  u32x4 o = raw;
  if (h < a.nq + a.nkv) {
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
      for (int k = 1; k < a.group; k <<= 1) ss += __shfl_xor(ss, k);
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
  const int slot = a.table[static_cast<size_t>(b) * a.max_pages + (static_cast<int>(pos) >> a.pt_shift)];
  if (static_cast<unsigned>(slot) >= static_cast<unsigned>(a.num_slots)) return;
  const bool is_k = h < a.nq + a.nkv;
  const int kvh = h - a.nq - (is_k ? 0 : a.nkv);
  const size_t at = ((static_cast<size_t>(slot) * a.nkv + kvh) << a.pt_shift) + off;
  if (is_k) {
    *reinterpret_cast<u32x4*>(a.k_pool + at * a.hd + d0) = o;
    return;
  }
  const int vb = a.pt_shift < 5 ? a.pt_shift : 5;
  uint16_t* v = a.v_pool + (((at >> vb) * a.hd + d0) << vb) + (off & ((1 << vb) - 1));
#pragma unroll
  for (int e = 0; e < 8; ++e)
    v[e << vb] = static_cast<uint16_t>(e & 1 ? o[e >> 1] >> 16 : o[e >> 1] & 0xffffu);
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
  VOOM_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim <= 256,
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
  a.group = 1;
  while (8 * a.group < head_dim) a.group <<= 1;
  a.pt_shift = ilog2(page_tokens);
  a.max_pages = max_pages;
  a.num_slots = num_slots;
  const long long total = static_cast<long long>(batch) * new_tokens *
                          (num_q_heads + 2LL * num_kv_heads) * a.group;
  VOOM_REQUIRE(total < (1LL << 38), "%s: too many heads in one call", who);
  hipLaunchKernelGGL(qk_norm_rope_append_kernel,
                     dim3(static_cast<unsigned>((total + kThreads - 1) / kThreads)), dim3(kThreads),
                     0, stream, a);
  return VOOM_LAUNCH_CHECK("qk_norm_rope_append: launch");
}
