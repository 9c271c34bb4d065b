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
// Keys are independent of each other, so nothing is merged: units of one stage (128
// tokens, 256 at D = 64) of all (sequence, kv head) segments lie end to end, as often as
// the window's rows go through the keys and after kLead that stand for what a segment costs
// besides, and are dealt out evenly (32 sequences of up to 4,000 tokens, 32/8 heads: 32 us,
// without kLead 61).  K goes straight into LDS (1 KiB loads) through a ring of four 32 KiB
// stages, three of them under way; loaded into operand registers instead, 64 bytes of
// a row at a time, the same keys took 147 us with no work on them, where 16 sequences of
// 1k-32k tokens, 32/8 heads, took 136 with all of it (118-129 since kLead).
//
// Eight wavefronts compute, RW of them on other rows (16 NT each, queries in registers)
// and 8 / RW on other keys of the stage:
//   scores[row][key] = Q . K^T   on v_mfma_f32_16x16x32_bf16, rows in the M dimension
// leaves a lane with four rows of one key, so that the sum over the rows needs one
// exchange per key tile.  A ninth wavefront adds the wavefronts' sums, one stage later,
// to the sums before and stores them: its loads and stores do not sit between the others'
// loads, which return in order.  Memory that is read and now and then written slows down:
// 16 sequences of 65,536 tokens, 32/8 heads, take 385 us, 5.75 TB/s, and without the stores
// 325; written eight stages at a time 368, but that takes registers from the kernels with
// more rows, and at D = 64 34 us became 36.
#include "paged_ring.h"

#include <cmath>

namespace voom {
namespace {

constexpr int kWaves = 8;                         // that compute
constexpr int kThreads = (kWaves + 1) * kWave;    // and the one that stores
constexpr int kLead = 3;                          // units that a segment costs besides its stages
constexpr int kMaxBatch = 1024;
constexpr int kStageElems = 128 * 128;
constexpr int stage_tokens(int D) { return kStageElems / D; }

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

__device__ __forceinline__ int window_of(const ObserveArgs& a, int b, int ctx) {
  int n = a.lens != nullptr ? a.lens[b] : a.L;
  n = n < 0 ? 0 : (n > a.L ? a.L : n);
  return n < ctx ? n : ctx;
}

// Chunk c (16 bytes) of K row r of a stage sits at c ^ k_swizzle(r) of its row: 16
// consecutive rows read one chunk each from 16 different 16-byte columns.
template <int D>
__device__ __forceinline__ int k_swizzle(int r) {
  return D == 128 ? (r & 15) : ((r >> 1) & 7);
}

// Starts this wavefront's loads of stage t (past the piece: empty ones, so that what is
// waited for does not depend on a branch).
template <int D>
__device__ __forceinline__ void load_stage(uint16_t* stage, const ObserveArgs& a, Pages& pg, int t,
                                           bool live, int wv, int lane) {
  constexpr int kBlocks = stage_tokens(D) / kBlk;
  constexpr int kPieces = kBlk * D / 512;  // of a block
  constexpr int kCpr = D / 8;              // 16-byte chunks of a row
  pg.hold(t * kBlocks, kBlocks, lane);
#pragma unroll
  for (int i = 0; i < kBlocks * kPieces / kWaves; ++i) {
    const int p = wv + kWaves * i;
    const int r = (p % kPieces) * (kWave / kCpr) + lane / kCpr;
    load_piece<2>(a.k_pool + pg.block(t * kBlocks + p / kPieces) * (kBlk * D),
                  live ? kBlk * D * 2 : 0,
                  r * (D * 2) + 16 * ((lane % kCpr) ^ k_swizzle<D>(r)), stage + p * 512);
  }
}

template <int D, int NT, int RW>
__global__ __launch_bounds__(kThreads) void gqa_observe_kernel(ObserveArgs a) {
  constexpr int kST = stage_tokens(D);
  constexpr int kRows = 16 * NT * RW;         // rows at a time
  constexpr int kKeys = kST / (kWaves / RW);  // a wavefront's keys of a stage
  // The ring: distinct objects, so that reads of one provably miss the pending loads of
  // the others.
  __shared__ __attribute__((aligned(1024))) uint16_t stage_0[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_1[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_2[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_3[kStageElems];
  __shared__ float part[2][RW][kST];  // a stage's sums of each group of rows
  static_assert(kStageElems * 2 / 1024 == 4 * kWaves, "the waits below count four loads a stage");

  const int lane = threadIdx.x & (kWave - 1);
  const int wv = uniform(threadIdx.x / kWave) & 15;
  const int i16 = lane & 15;
  const int g = lane >> 4;
  const int w = static_cast<int>(blockIdx.x);

  // This workgroup's units, found by every wavefront for itself.
  auto loads_of = [&](int b) {  // how often a sequence's keys are gone through
    if (a.L * a.G <= kRows) return 1;
    const int loads = (window_of(a, b, context_of(a, b)) * a.G + kRows - 1) / kRows;
    return loads < 1 ? 1 : loads;
  };
  auto units_of = [&](int b) {
    const int chunks = (context_of(a, b) + kST - 1) / kST;
    return chunks == 0 ? 0 : chunks * loads_of(b) + kLead;
  };
  int U = 0;
  for (int base = 0; base < a.B; base += kWave) {
    const int n = base + lane < a.B ? units_of(base + lane) * a.NKV : 0;
    U += __builtin_amdgcn_readlane(wave_inclusive_scan(n, lane), kWave - 1);
  }
  const Split split(U, a.W);
  if (w >= split.We || U == 0) return;
  int u0 = split.begin(w);
  const int u1 = split.begin(w + 1);
  int b = 0, units = 0, begin = 0;
  for (int base = 0;; base += kWave) {  // the sequence that holds unit u0
    const int n = base + lane < a.B ? units_of(base + lane) * a.NKV : 0;
    const int x = wave_inclusive_scan(n, lane);
    const int here = __builtin_amdgcn_readlane(x, kWave - 1);
    if (u0 < begin + here) {
      const int k = __popcll(__builtin_amdgcn_ballot_w64(begin + x <= u0));
      b = base + k;
      const int mine = __builtin_amdgcn_readlane(n, k);
      begin += __builtin_amdgcn_readlane(x, k) - mine;
      units = mine / a.NKV;
      break;
    }
    begin += here;
  }
  int kvh = (u0 - begin) / units;
  begin += kvh * units;

  while (true) {
    const int first = begin + kLead;  // the segment's first stage
    if (u1 <= first) return;
    const int loads = uniform(loads_of(b));
    int c0 = u0 > first ? u0 - first : 0;
    int c1 = (u1 < begin + units ? u1 : begin + units) - first;
    if (loads > 1) {
      c0 = (c0 + loads - 1) / loads;
      c1 = (c1 + loads - 1) / loads;
    }
    const int ctx = uniform(context_of(a, b));
    const int n = uniform(window_of(a, b, ctx));
    const int live = n * a.G;  // rows of the window, (token, head) with the head fastest
    const size_t out_row = (static_cast<size_t>(b) * a.NKV + kvh) * a.cap;

    for (int r0 = 0; c0 < c1 && (r0 == 0 || r0 < live); r0 += kRows) {
      if (wv == kWaves) {
        // the wavefront that stores: stage t - 1 while the others compute stage t
        const float* from = (r0 == 0 ? a.scores : a.out) + out_row;
        float old[kST / kWave];
        auto load_old = [&](int t) {
#pragma unroll
          for (int j = 0; j < kST / kWave; ++j) {
            const int p = t * kST + j * kWave + lane;
            old[j] = from[p < ctx ? p : ctx - 1];
          }
        };
        load_old(c0);
        lds_barrier();
        for (int t = c0; t < c1; ++t) {
          lds_barrier();  // stage t is computed
#pragma unroll
          for (int j = 0; j < kST / kWave; ++j) {
            float v = 0.f;
#pragma unroll
            for (int r = 0; r < RW; ++r) v += part[(t - c0) & 1][r][j * kWave + lane];
            const int p = t * kST + j * kWave + lane;
            if (p < ctx) a.out[out_row + p] = old[j] + v;
          }
          if (t + 1 < c1) load_old(t + 1);
        }
        continue;
      }
      const int rw = wv % RW;
      const int kw = wv / RW;
      // A operands of this wavefront's rows, their -lse in log2 units, and the last token
      // that each sees (-1: no row)
      u32x4 qa[NT][D / 32];
      f32x4 nl[NT];
      int vis[NT][4];
      bool some_dead = false;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int first = r0 + (rw * NT + i) * 16;
        const int r = first + i16 < live ? first + i16 : 0;
        const int tok = r / a.G;
        const int head = kvh * a.G + (r - tok * a.G);
        const uint16_t* qr =
            a.q + ((static_cast<size_t>(b) * a.NQ + head) * a.L + tok) * D + 8 * g;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) qa[i][s] = *reinterpret_cast<const u32x4*>(qr + 32 * s);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int re = first + 4 * g + e < live ? first + 4 * g + e : 0;
          const int te = re / a.G;
          const float v = a.lse[(static_cast<size_t>(b) * a.L + te) * a.NQ + kvh * a.G +
                                (re - te * a.G)];
          const bool none = v == -INFINITY || first + 4 * g + e >= live;
          nl[i][e] = none ? 0.f : v * -1.4426950408889634f;
          vis[i][e] = none ? -1 : ctx - n + te;
          some_dead |= none;
        }
      }
      const bool dead_rows = __builtin_amdgcn_ballot_w64(some_dead) != 0;
      const bool rows_here = r0 + rw * NT * 16 < live;

      Pages pg(a.table + static_cast<size_t>(b) * a.max_pages, a.max_pages, a.num_slots, a.NKV,
               kvh, a.pt_shift - 5, (ctx - 1) / kBlk);
      load_stage<D>(stage_0, a, pg, c0, true, wv, lane);
      load_stage<D>(stage_1, a, pg, c0 + 1, c0 + 1 < c1, wv, lane);
      load_stage<D>(stage_2, a, pg, c0 + 2, c0 + 2 < c1, wv, lane);
      int t = c0;
      // One stage: it has landed for every wavefront, and the one before is no longer read.
      auto step = [&](const uint16_t* cur, uint16_t* free) {
        // gfx9 encoding: vmcnt 8 (two stages), expcnt 7, lgkmcnt 15
        __builtin_amdgcn_s_waitcnt(0x0F78);
        lds_barrier();
        load_stage<D>(free, a, pg, t + 3, t + 3 < c1, wv, lane);
        const bool masked = dead_rows || (t + 1) * kST > ctx - n;
#pragma unroll 2
        for (int j = 0; j < kKeys / 16; ++j) {
          const int key = kw * kKeys + 16 * j + i16;  // of the stage
          float sum = 0.f;
          if (rows_here) {
            f32x4 sc[NT];
            u32x4 kb[D / 32];
#pragma unroll
            for (int s = 0; s < D / 32; ++s)
              kb[s] = *reinterpret_cast<const u32x4*>(cur + key * D +
                                                      8 * ((4 * s + g) ^ k_swizzle<D>(key)));
#pragma unroll
            for (int i = 0; i < NT; ++i) sc[i] = f32x4{};
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
#pragma unroll
              for (int i = 0; i < NT; ++i)
                sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, qa[i][s]), __builtin_bit_cast(bf16x8, kb[s]), sc[i],
                    0, 0, 0);
            }
            if (!masked) {
#pragma unroll
              for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  sum += fast_exp2(__builtin_fmaf(sc[i][e], a.scale, nl[i][e]));
              }
            } else {
#pragma unroll
              for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float x = fast_exp2(__builtin_fmaf(sc[i][e], a.scale, nl[i][e]));
                  sum += t * kST + key > vis[i][e] ? 0.f : x;
                }
              }
            }
            sum = wave_sum_across_groups(sum);
          }
          if (g == 0) part[(t - c0) & 1][rw][key] = sum;
        }
        return ++t < c1;
      };
      while (step(stage_0, stage_3) && step(stage_1, stage_0) && step(stage_2, stage_1) &&
             step(stage_3, stage_2)) {
      }
      wait_vmem_all();
      lds_barrier();  // the last stage is computed, the ring no longer read or written
    }
    u0 = u1 < begin + units ? u1 : begin + units;
    if (u0 >= u1) return;
    begin += units;
    if (++kvh == a.NKV) {
      kvh = 0;
      do {
        units = uniform(units_of(++b));
      } while (b < a.B - 1 && units == 0);
    }
  }
}

template <int D, int NT, int RW>
void launch_shape(const ObserveArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((gqa_observe_kernel<D, NT, RW>), dim3(static_cast<unsigned>(a.W)),
                     dim3(kThreads), 0, stream, a);
}

// As few wavefronts on other rows as hold them: the others then read other keys, and a
// key is read from LDS by fewer (131,072 tokens, 132 rows, 32/8 heads: NT = 2 on eight
// wavefronts 129 us, NT = 3 on four 90).
template <int D>
void launch_observe(const ObserveArgs& a, hipStream_t stream) {
  const int rows = a.L * a.G;
  if (rows <= 16) launch_shape<D, 1, 1>(a, stream);
  else if (rows <= 32) launch_shape<D, 2, 1>(a, stream);
  else if (rows <= 64) launch_shape<D, 2, 2>(a, stream);
  else if (rows <= 128) launch_shape<D, 4, 2>(a, stream);
  else if (rows <= 192) launch_shape<D, 3, 4>(a, stream);
  else launch_shape<D, 4, 4>(a, stream);
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
  const int st = stage_tokens(head_dim);
  const long long loads = (static_cast<long long>(window) * a.G + 255) / 256;
  const long long most =
      ((static_cast<long long>(max_pages) * page_tokens + st - 1) / st * loads + kLead) * batch *
      num_kv_heads;
  VOOM_REQUIRE(most < (1LL << 31), "%s: %d pages of %d tokens for %d sequences are too many", who,
               max_pages, page_tokens, batch);
  a.W = static_cast<int>(most < device_cu_count() ? most : device_cu_count());  // all run at once
  if (head_dim == 128) launch_observe<128>(a, stream);
  else launch_observe<64>(a, stream);
  return VOOM_LAUNCH_CHECK("paged_gqa_observe: launch");
}
