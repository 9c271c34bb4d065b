// Attention weight that cached tokens receive, for gfx950: the sums by which a
// bounded cache chooses what it keeps.
//
// The newest n = lens[b] of the ctx[b] cached tokens of sequence b are the window;
// its token t sees the tokens up to its own.  With the log-sum-exp of its scores
// (from the attention itself)
//   out[h][p] = scores[h][p] + sum_{t, heads g of kv head h} exp(scale q[t][g] . k[p] - lse[t][g])
// over the rows that see p, p < ctx.
//
// What bounds it: K of the context once (2 D bytes per token and kv head, 8 more for
// the sums) up to about 200 (token, head of the group) rows, then matrix work and an
// exponential per (row, key).
//
// Keys are independent of each other, so nothing is merged: the 256-token units of
// all (sequence, kv head) segments lie end to end and workgroup w of W takes
// [w U/W, (w+1) U/W).  The rows' queries (256 at a time) sit in LDS, a wavefront
// holds 64 keys in registers while the next 64 are under way, and
//   scores[row][key] = Q . K^T   on v_mfma_f32_16x16x32_bf16, rows in the M dimension
// leaves a lane with four rows of one key: the sum over the rows needs no exchange
// until the end of the unit.
#include "common.h"

#include <cmath>

namespace voom {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kBlk = 32;              // tokens of a K block in the pool
constexpr int kMine = 64;             // keys of a wavefront in a unit
constexpr int kUnit = kWaves * kMine;
constexpr int kRows = 256;            // rows in LDS at a time
constexpr int kMaxBatch = 1024;

struct ObserveArgs {
  const uint16_t* q;     // [B, NQ, L, D]
  const float* lse;      // [B, L, NQ]
  const uint16_t* k_pool;
  const int32_t* table;  // [B, max_pages]
  const int32_t* ctx;    // [B]
  const int32_t* lens;   // [B], or null: L each
  const float* scores;   // [B, NKV, cap]
  float* out;            // [B, NKV, cap]
  int B, NQ, NKV, G, L, cap, max_pages, pt_shift, num_slots;
  int W;                 // workgroups of the split
  float scale;           // softmax scale in log2 units
};

__device__ __forceinline__ int context_of(const ObserveArgs& a, int b) {
  int most = a.max_pages << a.pt_shift;
  most = most < a.cap ? most : a.cap;
  const int c = a.ctx[b];
  return c < 0 ? 0 : (c > most ? most : c);
}

template <int D>
struct Keys {
  u32x4 k[kMine / 16][D / 32];  // 16-key tiles x k-steps
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void gqa_observe_kernel(ObserveArgs a) {
  constexpr int kStride = D + 8;  // elements of a row in LDS: 16 rows start in 16 bank groups
  __shared__ int seg[kMaxBatch + 1];
  __shared__ int wave_tot[kWaves];
  __shared__ __attribute__((aligned(16))) uint16_t rows[kRows][kStride];
  __shared__ __attribute__((aligned(16))) float neg_lse[kRows];  // -lse in log2 units; -inf: no row

  const int lane = threadIdx.x & (kWave - 1);
  const int wv = uniform(threadIdx.x / kWave);
  const int i16 = lane & 15;
  const int g = lane >> 4;

  {  // exclusive prefix sum of the sequences' units
    int carry = 0;
    for (int base = 0; base < a.B; base += kThreads) {
      const int i = base + static_cast<int>(threadIdx.x);
      const int n = i < a.B ? (context_of(a, i) + kUnit - 1) / kUnit : 0;
      const int x = wave_inclusive_scan(n, lane);
      if (lane == kWave - 1) wave_tot[wv] = x;
      __syncthreads();
      int before = carry;
      for (int k = 0; k < wv; ++k) before += wave_tot[k];
      if (i < a.B) seg[i] = before + x - n;
      for (int k = 0; k < kWaves; ++k) carry += wave_tot[k];
      __syncthreads();
    }
    if (threadIdx.x == 0) seg[a.B] = carry;
    __syncthreads();
  }
  const long long U = static_cast<long long>(uniform(seg[a.B])) * a.NKV;
  const int We = static_cast<int>(U < a.W ? U : a.W);
  const int w = static_cast<int>(blockIdx.x);
  if (w >= We) return;
  long long u0 = static_cast<long long>(w) * U / We;
  const long long u1 = static_cast<long long>(w + 1) * U / We;
  int lo = 0, hi = a.B - 1;  // the sequence that holds unit u0
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (static_cast<long long>(uniform(seg[mid])) * a.NKV <= u0) lo = mid; else hi = mid - 1;
  }
  int b = lo;
  int units = uniform(seg[b + 1]) - uniform(seg[b]);
  long long begin = static_cast<long long>(uniform(seg[b])) * a.NKV;
  int kvh = static_cast<int>((u0 - begin) / units);
  begin += static_cast<long long>(kvh) * units;

  while (true) {
    const int c0 = static_cast<int>(u0 - begin);
    const int c1 = static_cast<int>((u1 < begin + units ? u1 : begin + units) - begin);
    const int ctx = uniform(context_of(a, b));
    int n = a.lens != nullptr ? uniform(a.lens[b]) : a.L;
    n = n < 0 ? 0 : (n > a.L ? a.L : n);
    n = n < ctx ? n : ctx;
    const int live = n * a.G;  // rows of the window, (token, head) with the head fastest
    const int32_t* trow = a.table + static_cast<size_t>(b) * a.max_pages;
    const size_t out_row = (static_cast<size_t>(b) * a.NKV + kvh) * a.cap;

    // a unit's keys of this wavefront: two 32-token blocks (past the context: the
    // last one again, not stored), the slots of 64 pages from win_page on in the lanes
    const int last_blk = (ctx - 1) / kBlk;
    const int sub_shift = a.pt_shift - 5;
    int win_page = -(1 << 30), win = 0;
    auto load_keys = [&](int c, Keys<D>& r) {
      int first = (c * kUnit + wv * kMine) / kBlk;
      first = first < last_blk ? first : last_blk;
      if (first >> sub_shift < win_page || (first + 1) >> sub_shift >= win_page + kWave) {
        win_page = first >> sub_shift;
        win = win_page + lane < a.max_pages ? trow[win_page + lane] : 0;
        wait_vmem_all();  // here, not at the readlanes below for every unit
      }
#pragma unroll
      for (int j = 0; j < kMine / kBlk; ++j) {
        int blk = first + j;
        blk = blk < last_blk ? blk : last_blk;
        const int page = blk >> sub_shift;
        int slot = __builtin_amdgcn_readlane(win, page - win_page);
        if (static_cast<unsigned>(slot) >= static_cast<unsigned>(a.num_slots)) slot = 0;
        const size_t at = ((static_cast<size_t>(slot) * a.NKV + kvh) << sub_shift) +
                          (blk - (page << sub_shift));
        const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(a.k_pool + at * (kBlk * D)), static_cast<short>(0),
            kBlk * D * 2, 0x00020000);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int s = 0; s < D / 32; ++s)
            r.k[2 * j + t][s] = __builtin_amdgcn_raw_buffer_load_b128(
                kr, (i16 * D + 8 * g) * 2 + (16 * t * D + 32 * s) * 2, 0, 2);
        }
      }
    };

    for (int r0 = 0; r0 == 0 || r0 < live; r0 += kRows) {
      const int here = live - r0 < kRows ? live - r0 : kRows;
      __syncthreads();  // the rows before are no longer read
      for (int idx = threadIdx.x; idx < ((here + 15) & ~15) * (D / 8); idx += kThreads) {
        const int r = idx / (D / 8);
        const int c = idx - r * (D / 8);
        u32x4 x = {0u, 0u, 0u, 0u};
        const int rr = r0 + r;
        const int t = rr / a.G;
        const int head = kvh * a.G + (rr - t * a.G);
        if (r < here)
          x = *reinterpret_cast<const u32x4*>(
              a.q + ((static_cast<size_t>(b) * a.NQ + head) * a.L + t) * D + 8 * c);
        *reinterpret_cast<u32x4*>(&rows[r][8 * c]) = x;
        if (c == 0) {
          const float v = r < here ? a.lse[(static_cast<size_t>(b) * a.L + t) * a.NQ + head]
                                   : -INFINITY;
          neg_lse[r] = v == -INFINITY ? -INFINITY : v * -1.4426950408889634f;
        }
      }
      __syncthreads();

      Keys<D> cur, nxt;
      load_keys(c0, cur);
      for (int c = c0; c < c1; ++c) {
        if (c + 1 < c1) load_keys(c + 1, nxt);
        const int first = c * kUnit + wv * kMine;
        const bool edge = first + kMine > ctx - n;  // some row may not see some key
        float sum[kMine / 16] = {};
        for (int i = 0; i < here; i += 16) {
          u32x4 qa[D / 32];
#pragma unroll
          for (int s = 0; s < D / 32; ++s)
            qa[s] = *reinterpret_cast<const u32x4*>(&rows[i + i16][32 * s + 8 * g]);
          const f32x4 nl = *reinterpret_cast<const f32x4*>(&neg_lse[i + 4 * g]);
          f32x4 sc[kMine / 16];
#pragma unroll
          for (int j = 0; j < kMine / 16; ++j) {
            sc[j] = f32x4{};
#pragma unroll
            for (int s = 0; s < D / 32; ++s)
              sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  __builtin_bit_cast(bf16x8, qa[s]), __builtin_bit_cast(bf16x8, cur.k[j][s]),
                  sc[j], 0, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool dead = nl[e] == -INFINITY;
            // the last token that the row sees
            const int vis = ctx - n + (edge ? (r0 + i + 4 * g + e) / a.G : n);
#pragma unroll
            for (int j = 0; j < kMine / 16; ++j) {
              const float x = fast_exp2(__builtin_fmaf(sc[j][e], a.scale, nl[e]));
              sum[j] += dead || first + 16 * j + i16 > vis ? 0.f : x;
            }
          }
        }
        // over the lane groups; group g then stores key tile g
        float mine = 0.f;
#pragma unroll
        for (int j = 0; j < kMine / 16; ++j) {
          const float v = wave_sum_across_groups(sum[j]);
          mine = g == j ? v : mine;
        }
        const int p = first + lane;
        if (p < ctx) {
          const float* from = r0 == 0 ? a.scores : a.out;
          a.out[out_row + p] = from[out_row + p] + mine;
        }
        cur = nxt;
      }
    }
    u0 = u1 < begin + units ? u1 : begin + units;
    if (u0 >= u1) return;
    begin += units;
    if (++kvh == a.NKV) {
      kvh = 0;
      do {
        ++b;
      } while (b < a.B - 1 && uniform(seg[b + 1]) == uniform(seg[b]));
      units = uniform(seg[b + 1]) - uniform(seg[b]);
    }
  }
}

}  // namespace
}  // namespace voom

using namespace voom;

extern "C" int voom_paged_gqa_observe(const void* q, const float* lse, const void* k_pool,
                                      const int32_t* block_table, const int32_t* ctx_lens,
                                      const int32_t* window_lens, const float* scores, float* out,
                                      int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                      int page_tokens, int max_pages, int num_slots, int window,
                                      int score_tokens, float scale, hipStream_t stream) {
  const char* who = "paged_gqa_observe";
  VOOM_REQUIRE(q && lse && k_pool && block_table && ctx_lens && scores && out,
               "%s: null pointer argument", who);
  VOOM_REQUIRE(num_slots > 0, "%s: empty page pool", who);
  VOOM_REQUIRE(batch > 0 && batch <= kMaxBatch && num_kv_heads > 0 && num_q_heads > 0 &&
                   num_q_heads % num_kv_heads == 0 && (head_dim == 64 || head_dim == 128) &&
                   window > 0 && max_pages > 0 &&
                   static_cast<long long>(batch) * num_q_heads * window < (1LL << 28),
               "%s: unsupported geometry (batch %d, heads %d/%d, head_dim %d, window %d)", who,
               batch, num_q_heads, num_kv_heads, head_dim, window);
  VOOM_REQUIRE(is_pow2(page_tokens) && page_tokens >= 32 && page_tokens <= 4096,
               "%s: page_tokens %d must be a power of two in [32, 4096]", who, page_tokens);
  VOOM_REQUIRE(static_cast<long long>(max_pages) * page_tokens < (1LL << 30),
               "%s: block table of %d pages of %d tokens", who, max_pages, page_tokens);
  VOOM_REQUIRE(score_tokens > 0, "%s: no room for scores", who);
  VOOM_REQUIRE(std::isfinite(scale), "%s: the scale must be finite", who);
  VOOM_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(k_pool) % 16 == 0,
               "%s: q and the pool must be 16-byte aligned", who);
  ObserveArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.lse = lse;
  a.k_pool = static_cast<const uint16_t*>(k_pool);
  a.table = block_table;
  a.ctx = ctx_lens;
  a.lens = window_lens;
  a.scores = scores;
  a.out = out;
  a.B = batch;
  a.NQ = num_q_heads;
  a.NKV = num_kv_heads;
  a.G = num_q_heads / num_kv_heads;
  a.L = window;
  a.cap = score_tokens;
  a.max_pages = max_pages;
  a.pt_shift = ilog2(page_tokens);
  a.num_slots = num_slots;
  a.scale = scale * 1.4426950408889634f;
  const long long most = static_cast<long long>(batch) * num_kv_heads *
                         ((static_cast<long long>(max_pages) * page_tokens + kUnit - 1) / kUnit);
  a.W = static_cast<int>(most < 2LL * device_cu_count() ? most : 2LL * device_cu_count());
  const dim3 grid(static_cast<unsigned>(a.W));
  if (head_dim == 128)
    hipLaunchKernelGGL(gqa_observe_kernel<128>, grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL(gqa_observe_kernel<64>, grid, dim3(kThreads), 0, stream, a);
  return VOOM_LAUNCH_CHECK("paged_gqa_observe: launch");
}
