// The norm behind a block, the residual add and the norm before the next block, for gfx950:
//   y = x + scale * gate * post_weight * delta / sqrt(mean delta^2 + eps)
//   out = weight * y / sqrt(mean y^2 + eps)
// y becomes the residual stream (in place or in another buffer), out the next block's
// input.  All of it in fp32, y and out rounded to bf16 once each; out is formed of the
// unrounded y.
//
// What bounds it: x and delta read and y and out written once, 8 bytes an element; for few
// rows the launch and two sums, one after the other.  A row stays in registers between them,
// 8 dims a chunk: one wavefront a row up to kWaveDims dims, else a workgroup.  6,006 rows of
// 4,096: 42 us, 4.7 TB/s of reads and stores; one row of 576: 2.5 us.
#include "common.h"

namespace voom {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunks = 4;                     // chunks of 8 dims that a lane holds
constexpr int kWaveDims = 8 * kChunks * kWave;  // of a row that one wavefront holds
constexpr int kMaxHidden = kWaves * kWaveDims;

struct PostArgs {
  const uint16_t* x;       // [rows, hidden]
  const uint16_t* delta;
  const uint16_t* post_weight;  // [hidden]
  const uint16_t* weight;
  const uint16_t* gate;    // [rows / gate_rows, hidden], or null
  uint16_t* x_out;
  uint16_t* out;
  int rows, hidden, gate_rows;
  float eps, scale;
};

__device__ __forceinline__ void unpack8(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = __builtin_bit_cast(float, v[e] << 16);
    f[2 * e + 1] = __builtin_bit_cast(float, v[e] & 0xffff0000u);
  }
}

__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
               pack_bf16x2(f[6], f[7])};
}

// LANES: lanes that share a row, a wavefront's or the workgroup's.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* shared) {
  v = wave_sum_uniform(v);
  if constexpr (LANES == kWave) return v;
  if ((threadIdx.x & (kWave - 1)) == 0) shared[threadIdx.x / kWave] = v;
  __syncthreads();
  return (shared[0] + shared[1]) + (shared[2] + shared[3]);
}

template <int LANES>
__global__ __launch_bounds__(kThreads) void add_post_norm_kernel(PostArgs a) {
  __shared__ float sums[2][kWaves];
  const int lane = static_cast<int>(threadIdx.x) & (LANES - 1);
  const int row = LANES == kWave
                      ? static_cast<int>(blockIdx.x) * kWaves + uniform(threadIdx.x / kWave)
                      : static_cast<int>(blockIdx.x);
  if (row >= a.rows) return;  // (a whole wavefront; with a workgroup per row none)
  const size_t at = static_cast<size_t>(row) * a.hidden;
  const uint16_t* gate =
      a.gate != nullptr ? a.gate + static_cast<size_t>(row / a.gate_rows) * a.hidden : nullptr;
  const int chunks = a.hidden / 8;
  u32x4 d[kChunks], x[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = lane + i * LANES;
    if (c < chunks) {
      d[i] = *reinterpret_cast<const u32x4*>(a.delta + at + 8 * c);
      x[i] = *reinterpret_cast<const u32x4*>(a.x + at + 8 * c);
    } else {
      d[i] = u32x4{};
      x[i] = u32x4{};
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    float f[8];
    unpack8(d[i], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[e], f[e], ss);
  }
  const float n = static_cast<float>(a.hidden);
  const float r = a.scale / sqrtf(row_sum<LANES>(ss, sums[0]) / n + a.eps);
  float y[kChunks][8];
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = lane + i * LANES;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[i][e] = 0.f;
    if (c >= chunks) continue;
    float w[8], f[8], u[8];
    unpack8(*reinterpret_cast<const u32x4*>(a.post_weight + 8 * c), w);
    if (gate != nullptr) {
      unpack8(*reinterpret_cast<const u32x4*>(gate + 8 * c), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] *= f[e];
    }
    unpack8(d[i], f);
    unpack8(x[i], u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[i][e] = __builtin_fmaf(f[e] * r, w[e], u[e]);
      ss = __builtin_fmaf(y[i][e], y[i][e], ss);
    }
    *reinterpret_cast<u32x4*>(a.x_out + at + 8 * c) = pack8(y[i]);
  }
  const float q = 1.f / sqrtf(row_sum<LANES>(ss, sums[1]) / n + a.eps);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = lane + i * LANES;
    if (c >= chunks) continue;
    float w[8];
    unpack8(*reinterpret_cast<const u32x4*>(a.weight + 8 * c), w);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * q * w[e];
    *reinterpret_cast<u32x4*>(a.out + at + 8 * c) = pack8(y[i]);
  }
}

}  // namespace
}  // namespace voom

using namespace voom;

extern "C" int voom_add_post_norm(const void* x, const void* delta, const void* post_weight,
                                  const void* weight, const void* gate, int gate_rows, void* x_out,
                                  void* out, int rows, int hidden, float eps, float scale,
                                  hipStream_t stream) {
  const char* who = "add_post_norm";
  VOOM_REQUIRE(x && delta && post_weight && weight && x_out && out, "%s: null pointer argument",
               who);
  VOOM_REQUIRE(rows > 0 && hidden > 0 && hidden % 8 == 0 && hidden <= kMaxHidden,
               "%s: %d rows of hidden %d, which must be a multiple of 8 up to %d", who, rows,
               hidden, kMaxHidden);
  VOOM_REQUIRE(gate == nullptr || (gate_rows > 0 && rows % gate_rows == 0),
               "%s: a gate for every %d of %d rows", who, gate_rows, rows);
  VOOM_REQUIRE(eps >= 0.f, "%s: eps must not be negative", who);
  for (const void* p : {x, delta, post_weight, weight, gate, static_cast<const void*>(x_out),
                        static_cast<const void*>(out)})
    VOOM_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "%s: tensors must be 16-byte aligned",
                 who);
  PostArgs a;
  a.x = static_cast<const uint16_t*>(x);
  a.delta = static_cast<const uint16_t*>(delta);
  a.post_weight = static_cast<const uint16_t*>(post_weight);
  a.weight = static_cast<const uint16_t*>(weight);
  a.gate = static_cast<const uint16_t*>(gate);
  a.x_out = static_cast<uint16_t*>(x_out);
  a.out = static_cast<uint16_t*>(out);
  a.rows = rows;
  a.hidden = hidden;
  a.gate_rows = gate_rows;
  a.eps = eps;
  a.scale = scale;
  if (hidden <= kWaveDims)
    hipLaunchKernelGGL(add_post_norm_kernel<kWave>,
                       dim3(static_cast<unsigned>((rows + kWaves - 1) / kWaves)), dim3(kThreads),
                       0, stream, a);
  else
    hipLaunchKernelGGL(add_post_norm_kernel<kThreads>, dim3(static_cast<unsigned>(rows)),
                       dim3(kThreads), 0, stream, a);
  return VOOM_LAUNCH_CHECK("add_post_norm: launch");
}
