// Paged GQA attention of ragged chunks for gfx950: the newest tokens of each sequence (one
// of a running request, a part of a prompt, a whole prompt) over the paged K/V cache.
//
// Sequence b holds ctx[b] tokens, the newest n of them with queries.  The token at i scores
// the one at j
//   s = scale q.k,  with a cap c:  s = c tanh(s / c),  with slopes:  s -= slope[head] |i - j|
// and sees it where (j <= i and i - j < window) or j < prefix[b]:
//   out = sum_j softmax_j(s) v[j],  lse = log sum_j exp s.
// Rows that see nothing give 0 and -inf.
//
// What bounds it: K and V of the tokens seen once (4 D bytes per token and kv head) while
// few rows share them, then matrix work, 4 NQ D flops per (new token, token seen).
//
// gqa_chunk_rows_kernel, for small calls of many rows (kind_of; single tokens:
// gqa_chunk_token.hip, long ones: gqa_chunk_wide.hip), is built as gqa_tree_kernel is
// (paged_rows.h): a workgroup takes 64 rows (new token, head of the group) of a (sequence, kv
// head); the stages of 64 tokens (128 at D = 64) that a sequence's rows see, those behind the
// prefix and before the window left out, are the units of its segments, which lie end to end
// and are dealt out evenly; gqa_chunk_reduce_kernel merges cut ones.  Stages run through one
// ring in order; a stage that every row of the tile sees whole skips the masks.  8 sequences of
// 16,000 tokens, 32 rows, 8 kv heads of 128: 107 us, K and V at 4.9 TB/s.
#include "chunk_few.h"

#include <climits>

namespace voom {
namespace {

constexpr int kRows = 16 * kRowWaves;  // of a tile
template <int D>
using Geo = Geometry<kRows, stage_tokens(D), 8, 1>;

// A block that some row of the tile does not see whole.
template <int D>
__device__ __forceinline__ void edge_block(const uint16_t* tile, const u32x4 (&qop)[1][D / 32],
                                           const ChunkArgs& a, State<D, 1>& st, const View& view,
                                           int bi, int lane) {
  const int pos = bi * kBlk + 8 * (lane >> 4);
  f32x4 sc[1][2];
  u32x4 p[1];
  {
    Operands<D> o;
    read_keys<D>(o, tile, lane);
    scores_of<D, 1>(o, qop, sc);
  }
  score(sc, a, view, pos);
  const uint32_t seen = view.seen(pos);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    sc[0][e >> 2][e & 3] = (seen >> e & 1) != 0 ? sc[0][e >> 2][e & 3] : -INFINITY;
  weights_of<D>(sc, st, p);
  masked_products<D, 1>([&](int n) { return read_v<D>(tile, n, lane); }, p, st, view.ctx - pos,
                        [&](int) { return seen; });
}

template <int D, int AUX>
__global__ __launch_bounds__(kThreads, 2) void gqa_chunk_rows_kernel(ChunkArgs a) {
  constexpr int kBlocks = stage_blocks(D);
  constexpr int kTok = stage_tokens(D), kLead = Geo<D>::kLead;
  constexpr int kLoads = 2 * kBlocks * (kBlk * D / 512) / kWaves;  // a wavefront's, of a stage
  constexpr int kPad = D + 4;  // floats of a row in LDS: 16 rows start in 16 bank groups
  // The ring.  Distinct objects, so that reads of one provably miss the pending
  // direct-to-LDS loads of the others; the merge uses them when the loop is done.
  __shared__ __attribute__((aligned(1024))) uint16_t stage_0[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_1[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_2[kStageElems];
  __shared__ __attribute__((aligned(1024))) uint16_t stage_3[kStageElems];
  static_assert(kLoads == 4, "the waits below count the loads of a stage");
  static_assert(sizeof(float) * 16 * kPad <= sizeof(stage_0), "a merge buffer fits a stage");

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

  int b = 0, kvh, tile, c0, c1, chunks = 0, tiles = 1, pre = 0, gap = 0;
  int u0 = w, u1 = w + 1, begin = 0;  // the workgroup's units, and the segment's first one
  int x0;  // (every wavefront for itself: no barrier)
  const Units<Geo<D>> first = scan_units<Geo<D>>(a, 0, lane, x0);
  if (a.W != 0) {
    int U = __builtin_amdgcn_readlane(x0, kWave - 1);
    for (int base = kWave; base < a.B; base += kWave) {
      int x;
      scan_units<Geo<D>>(a, base, lane, x);
      U += __builtin_amdgcn_readlane(x, kWave - 1);
    }
    const Split split = split_of<Geo<D>>(U, a.W);
    if (w >= split.We || U == 0) return;
    u0 = split.begin(w);
    u1 = split.begin(w + 1);
  }
  for (int base = 0;; base += kWave) {  // the sequence that holds unit u0
    if (base >= a.B) return;
    int x = x0;
    Units<Geo<D>> units = first;
    if (base != 0) units = scan_units<Geo<D>>(a, base, lane, x);
    const int here = __builtin_amdgcn_readlane(x, kWave - 1);
    if (u0 < begin + here) {
      const int k = __popcll(__builtin_amdgcn_ballot_w64(begin + x <= u0));
      b = base + k;
      chunks = __builtin_amdgcn_readlane(units.chunks, k);
      tiles = __builtin_amdgcn_readlane(units.tiles, k);
      pre = __builtin_amdgcn_readlane(units.pre, k);
      gap = __builtin_amdgcn_readlane(units.gap, k);
      begin += __builtin_amdgcn_readlane(x, k) - __builtin_amdgcn_readlane(units.all(a), k);
      break;
    }
    begin += here;
  }
  {
    const int each = a.W != 0 ? chunks + kLead : 1;
    const int s = (u0 - begin) / each;
    kvh = s / tiles;
    tile = s - kvh * tiles;
    begin += s * each;
  }
  while (true) {
    if (a.W == 0) {
      c0 = 0;
      c1 = chunks;  // (0 below for a tile behind a padded sequence's new tokens)
    } else {
      const int at = begin + kLead;  // the segment's first stage
      if (u1 <= at) return;
      c0 = u0 > at ? u0 - at : 0;
      c1 = (u1 < at + chunks ? u1 : at + chunks) - at;
    }
    const int ctx = uniform(context_of(a, b));
    int base;
    const int n = uniform(new_of(a, b, base));
    const int prefix = uniform(prefix_of(a, b, ctx));
    if (tile * kRows >= n * a.G) c1 = c0;
    // the row of this lane's column, and what the tile's rows all see
    const int row = tile * kRows + rw * 16 + i16;
    const int t_row = row / a.G;
    const bool live = t_row < n;
    const int head = kvh * a.G + (row - t_row * a.G);
    View view;
    {
      const Sight sight(a, ctx, n, prefix, t_row);
      view.ctx = ctx;
      view.pre = live ? prefix : 0;
      view.at = sight.at;
      view.lo = sight.lo;
      view.hi = live ? sight.hi : 0;
      view.biased = a.slopes != nullptr;
      view.slope = view.biased ? a.slopes[head] * 1.4426950408889634f : 0.f;
    }
    const int t_lo = tile * kRows / a.G;
    int t_hi = (tile * kRows + kRows - 1) / a.G;
    t_hi = t_hi < n ? t_hi : n - 1;
    const int hi_min = Sight(a, ctx, n, prefix, t_lo).hi;
    const int lo_max = Sight(a, ctx, n, prefix, t_hi).lo;
    // Q^T operands of this wavefront's rows
    u32x4 qop[1][D / 32];
    {
      const uint16_t* qr = a.q + (live ? query_at(a, b, base, t_row, head) * D : 0) + 8 * g;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) qop[0][s] = *reinterpret_cast<const u32x4*>(qr + 32 * s);
    }
    State<D, 1> st;
    // never -inf: keys of score -inf then weigh 0 also where nothing came before
    st.m[0] = -FLT_MAX;
    st.l[0] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.acc[0][i] = f32x4{};

    const int last_blk = (ctx - 1) / kBlk;
    Pages pg(a.table + static_cast<size_t>(b) * a.max_pages, a.max_pages, a.num_slots, a.NKV, kvh,
             a.pt_shift - 5, last_blk);
    // (else this wavefront only loads)
    const bool rows_here = tile * kRows + rw * 16 < n * a.G;
    int t = c0;
    auto stage_of = [&](int c) { return c < pre ? c : c + gap; };
    auto load = [&](int c, uint16_t* stage) {
      load_stage<D, AUX>(stage, a.k_pool, a.v_pool, pg, stage_of(c) * kBlocks, wv, lane);
    };
    if (t < c1) load(t, stage_0);
    if (t + 1 < c1) load(t + 1, stage_1);
    if (t + 2 < c1) load(t + 2, stage_2);
    auto step = [&](const uint16_t* cur, uint16_t* free) {
      // Stage t has landed for every wavefront, and stage t - 1 is no longer read.  gfx9
      // encoding: vmcnt of the loads of stages t + 1 and t + 2, expcnt 7, lgkmcnt 15.
      if (t + 2 < c1) __builtin_amdgcn_s_waitcnt(0x0F78);
      else if (t + 1 < c1) __builtin_amdgcn_s_waitcnt(0x0F74);
      else __builtin_amdgcn_s_waitcnt(0x0F70);
      lds_barrier();
      const int at = stage_of(t) * kTok;
      if ((at >= lo_max && at + kTok <= hi_min) || at + kTok <= prefix) {
        Operands<D> o;  // (the next loads are prepared while the first operands come)
        read_block<D>(o, cur + kw * block_elems(D), lane);
        if (t + 3 < c1) load(t + 3, free);
#pragma unroll
        for (int j = 0; j < kBlocks / kKeyWaves && rows_here; ++j) {
          if (j != 0) read_block<D>(o, cur + (kKeyWaves * j + kw) * block_elems(D), lane);
          f32x4 sc[1][2];
          u32x4 p[1];
          scores_of<D, 1>(o, qop, sc);
          score(sc, a, view, at + (kKeyWaves * j + kw) * kBlk + 8 * g);
          weights_of<D>(sc, st, p);
          products<D, 1>(o, p, st);
        }
      } else {
        if (t + 3 < c1) load(t + 3, free);
        if (rows_here) {
#pragma unroll 1
          for (int j = kw; j < kBlocks && at / kBlk + j <= last_blk; j += kKeyWaves)
            edge_block<D>(cur + j * block_elems(D), qop, a, st, view, at / kBlk + j, lane);
        }
      }
      return ++t < c1;
    };
    if (t < c1) {
      while (step(stage_0, stage_3) && step(stage_1, stage_0) && step(stage_2, stage_1) &&
             step(stage_3, stage_2)) {
      }
    }
    wait_vmem_all();
    lds_barrier();  // the ring is no longer read or written

    // Merge the two wavefronts of each group of rows: one leaves its state in LDS, the
    // other adds its own and writes.
    const bool all = a.W == 0 || (c0 == 0 && c1 == chunks);
    const size_t slot = 2 * static_cast<size_t>(w) + (c0 == 0 ? 1 : 0);
    float* const buf = reinterpret_cast<float*>(rw < 2 ? (rw == 0 ? stage_0 : stage_1)
                                                       : (rw == 2 ? stage_2 : stage_3)) +
                       i16 * kPad;
    const float lt = wave_sum_across_groups(st.l[0]);
    if (kw == 1) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<f32x4*>(buf + 16 * i + 4 * g) = st.acc[0][i];
      if (g == 0) {
        buf[D] = st.m[0];
        buf[D + 1] = lt;
      }
    }
    __syncthreads();
    if (kw == 0) {
      const float m1 = buf[D];
      const float M = fmaxf(st.m[0], m1);
      const float f0 = fast_exp2(st.m[0] - M), f1 = fast_exp2(m1 - M);
      const float L = lt * f0 + buf[D + 1] * f1;
      const bool empty = !live || L == 0.f;
      const float inv = 1.f / L;
      const int r = rw * 16 + i16;
      // (rows behind the last one are in the workspace, but not in out)
      const bool mine = a.starts != nullptr ? live : t_row < a.T;
      const size_t at = out_at(a, b, base, t_row, head);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const f32x4 o =
            st.acc[0][i] * f0 + *reinterpret_cast<const f32x4*>(buf + 16 * i + 4 * g) * f1;
        if (!all) {
          *reinterpret_cast<f32x4*>(a.part_o + (slot * kRows + r) * D + 16 * i + 4 * g) = o;
        } else if (mine) {
          *reinterpret_cast<u32x2*>(a.out + at * D + 16 * i + 4 * g) =
              empty ? u32x2{0u, 0u}
                    : u32x2{pack_bf16x2(o[0] * inv, o[1] * inv),
                            pack_bf16x2(o[2] * inv, o[3] * inv)};
        }
      }
      if (g == 0 && !all) *reinterpret_cast<float2*>(a.part_ml + (slot * kRows + r) * 2) = {M, L};
      if (g == 0 && all && mine && a.lse != nullptr)
        a.lse[at] = empty ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
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
          const Units<Geo<D>> units(a, ++b);
          chunks = uniform(units.chunks);
          tiles = uniform(units.tiles);
          pre = uniform(units.pre);
          gap = uniform(units.gap);
        } while (b < a.B - 1 && chunks == 0);
      }
    }
    __syncthreads();  // the next piece writes the ring
  }
}

constexpr int kShort = 8;  // stages of a segment that is not cut

FewPlan plan_rows(int B, int NKV, int D, int G, int N, int T, long long tokens, int window) {
  FewPlan p;
  const long long tok = stage_tokens(D);
  const long long tiles = N > 0 ? static_cast<long long>(N) * G / kRows + (B < N ? B : N)
                                : static_cast<long long>(B) * ((T * G + kRows - 1) / kRows);
  p.segs = tiles * NKV;
  long long stages = (tokens + tok - 1) / tok;
  const long long seen = (static_cast<long long>(window) + kRows / G) / tok + 2;
  if (seen < stages) stages = seen;
  // All workgroups of a split run at once.  Without one a workgroup walks a segment, which
  // saves the merges and the reduce launch, where the segments are short, the longer if they
  // fill half of the card (32 rows, 8 kv heads of 128; without and with the split: 8 segments of
  // 500 tokens 14.6 and 14.5 us, of 1,000 21.9 and 14.3; 256 of 1,000 29.6 and 34.9).
  const int cus = device_cu_count();
  const long long full = (p.segs + cus - 1) / cus * cus;
  const int most = 2 * p.segs >= full ? 2 * kShort : kShort;
  p.W = stages <= most ? 0 : cus;
  p.rows = kRows;
  return p;
}

// The kernel that takes a call goes by its rows (new token, head of the group) a kv head.  All
// three are right for any lengths.
//
// Up to 16 rows a sequence: that of single tokens, since it streams K and V fastest.  It reads
// them once for every 16 rows, though, so that packed rows, one chunk among many single tokens
// perhaps, are two a sequence at most on the average.  64 sequences of 500 to 4,000 tokens, 32/8
// heads of 128, in us, it and the one of long chunks:
//   2 tokens each  98  132    63 single tokens and a chunk of 64  138  143    of 128  178  142
//
// Beyond that the one of long chunks, which cuts and orders its work by lengths (64 such
// sequences of 8 tokens: 135 us, the one above 201; 16 tokens: 138 and 315).  It has three
// launches and longer ones, 30 us at least where the one above has 15: small calls take that
// (32/8 heads, 300 rows a kv head of 1,000 to 1,200 tokens: 23 us against 38; of 8,100 tokens:
// 51 against 44.  9/3 heads of 64, 16 sequences, 8 tokens each: 18 and 24; one chunk of 256:
// 29 and 27).
enum class Kind { kToken, kRows, kWide };
constexpr long long kSmall = 1LL << 22;  // rows times the tokens of 128 dims that they may see
Kind kind_of(int batch, int rows, int tokens, int NKV, int G, int D, long long cap, int window) {
  const long long all = rows > 0 ? static_cast<long long>(rows) * G
                                 : static_cast<long long>(tokens) * G * batch;
  const long long reach = window > 0 ? static_cast<long long>(window) + rows + tokens : cap;
  const long long seen = reach < cap ? reach : cap;
  const bool small = all <= kSmall * (128 / D) / (seen * NKV);
  if (all <= 16LL * batch && (rows <= 2 * batch || small)) return Kind::kToken;
  return small ? Kind::kRows : Kind::kWide;
}

FewPlan plan_few(Kind kind, int B, int NKV, int D, int G, int N, int T, long long tokens,
                 int window) {
  return kind == Kind::kToken ? plan_token(B, NKV, D, G, N, T, tokens, window)
                              : plan_rows(B, NKV, D, G, N, T, tokens, window);
}

bool chunk_shape_ok(int batch, int rows, int tokens, int num_q_heads, int num_kv_heads,
                    int head_dim, int page_tokens, int max_pages) {
  const long long all = rows > 0 ? rows : static_cast<long long>(batch) * tokens;
  return batch > 0 && batch <= kMaxChunkBatch && (rows > 0) != (tokens > 0) && rows >= 0 &&
         tokens >= 0 && num_kv_heads > 0 && num_kv_heads <= 65535 && num_q_heads > 0 &&
         num_q_heads % num_kv_heads == 0 && num_q_heads / num_kv_heads <= 16 &&
         (head_dim == 64 || head_dim == 128) && is_pow2(page_tokens) && page_tokens >= 32 &&
         page_tokens <= 4096 && max_pages > 0 &&
         static_cast<long long>(max_pages) * page_tokens < (1LL << 30) &&
         all * num_q_heads < (1LL << 28);
}

size_t part_o_bytes(const FewPlan& p, int D) {
  return static_cast<size_t>(2) * p.W * p.rows * D * sizeof(float);
}

}  // namespace
}  // namespace voom

using namespace voom;

extern "C" size_t voom_paged_gqa_chunk_workspace_bytes(int batch, int rows, int tokens,
                                                       int num_q_heads, int num_kv_heads,
                                                       int head_dim, int page_tokens,
                                                       int max_pages, int window) {
  if (!chunk_shape_ok(batch, rows, tokens, num_q_heads, num_kv_heads, head_dim, page_tokens,
                      max_pages) || window < 0)
    return 0;
  const int G = num_q_heads / num_kv_heads;
  const long long cap = static_cast<long long>(max_pages) * page_tokens;
  const Kind kind = kind_of(batch, rows, tokens, num_kv_heads, G, head_dim, cap, window);
  if (kind == Kind::kWide)
    return plan_wide(batch, num_kv_heads, head_dim, G, rows, tokens, cap).bytes;
  const FewPlan p = plan_few(kind, batch, num_kv_heads, head_dim, G, rows, tokens, cap,
                             window == 0 ? INT_MAX : window);
  return part_o_bytes(p, head_dim) + static_cast<size_t>(2) * p.W * p.rows * 2 * sizeof(float);
}

extern "C" int voom_paged_gqa_chunk(const void* q, const void* k_pool, const void* v_pool,
                                    const int32_t* block_table, const int32_t* ctx_lens,
                                    const int32_t* starts, const int32_t* new_lens,
                                    const float* slopes, const int32_t* prefix_lens, void* out,
                                    float* lse, void* workspace, size_t ws_bytes, int batch,
                                    int rows, int tokens, int num_q_heads, int num_kv_heads,
                                    int head_dim, int page_tokens, int max_pages, int num_slots,
                                    int window, float scale, float softcap, hipStream_t stream) {
  const char* who = "paged_gqa_chunk";
  VOOM_REQUIRE(q && k_pool && v_pool && block_table && ctx_lens && out,
               "%s: null pointer argument", who);
  VOOM_REQUIRE(num_slots > 0, "%s: empty page pool", who);
  VOOM_REQUIRE(chunk_shape_ok(batch, rows, tokens, num_q_heads, num_kv_heads, head_dim,
                              page_tokens, max_pages),
               "%s: unsupported geometry (batch %d, %d rows, %d tokens, heads %d/%d, head_dim %d, "
               "%d pages of %d)",
               who, batch, rows, tokens, num_q_heads, num_kv_heads, head_dim, max_pages,
               page_tokens);
  VOOM_REQUIRE((starts != nullptr) == (rows > 0) && (starts == nullptr || new_lens == nullptr),
               "%s: packed rows come with starts, padded ones with new_lens", who);
  VOOM_REQUIRE(window >= 0, "%s: window %d must not be negative", who, window);
  VOOM_REQUIRE(std::isfinite(scale) && std::isfinite(softcap) && softcap >= 0.f,
               "%s: the scale must be finite, the cap finite and not negative", who);
  // (the cap's polynomial has coefficients up to scale (scale / softcap)^6)
  const float cap_k = softcap > 0.f ? scale / softcap : 0.f;
  const float cap_k2 = cap_k * cap_k;
  VOOM_REQUIRE(cap_k == 0.f ? softcap == 0.f || scale == 0.f
                            : std::isnormal(cap_k) && std::isfinite(2.f * softcap) &&
                                  std::isfinite(2.f * scale * cap_k2 * cap_k2 * cap_k2),
               "%s: a cap of %g is out of proportion to a scale of %g", who,
               static_cast<double>(softcap), static_cast<double>(scale));
  VOOM_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(k_pool) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(v_pool) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 8 == 0,
               "%s: q and pools must be 16-byte aligned", who);
  const int G = num_q_heads / num_kv_heads;
  const int win = window == 0 ? INT_MAX : window;
  const long long cap = static_cast<long long>(max_pages) * page_tokens;
  const Kind kind = kind_of(batch, rows, tokens, num_kv_heads, G, head_dim, cap, window);
  const FewPlan p = plan_few(kind, batch, num_kv_heads, head_dim, G, rows, tokens, cap, win);
  VOOM_REQUIRE(kind == Kind::kWide || (cap / kBlk + 16) * p.segs < (1LL << 31),
               "%s: %d pages of %d tokens for %d sequences are too many", who, max_pages,
               page_tokens, batch);
  const size_t need = voom_paged_gqa_chunk_workspace_bytes(batch, rows, tokens, num_q_heads,
                                                           num_kv_heads, head_dim, page_tokens,
                                                           max_pages, window);
  VOOM_REQUIRE(need == 0 || (workspace != nullptr && ws_bytes >= need &&
                             reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
               "%s: workspace %zu bytes < required %zu (16-byte aligned)", who, ws_bytes, need);
  ChunkArgs a;
  a.q = static_cast<const uint16_t*>(q);
  a.k_pool = static_cast<const uint16_t*>(k_pool);
  a.v_pool = static_cast<const uint16_t*>(v_pool);
  a.table = block_table;
  a.ctx = ctx_lens;
  a.starts = starts;
  a.lens = new_lens;
  a.slopes = slopes;
  a.prefix = prefix_lens;
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.B = batch;
  a.NQ = num_q_heads;
  a.NKV = num_kv_heads;
  a.G = G;
  a.T = tokens;
  a.N = rows;
  a.max_pages = max_pages;
  a.pt_shift = ilog2(page_tokens);
  a.num_slots = num_slots;
  a.window = win;
  a.scale = scale * 1.4426950408889634f;
  a.cap = softcap * 1.4426950408889634f;
  a.cap_k = cap_k;
  a.part_o = a.part_ml = nullptr;
  a.W = a.per_xcd = 0;
  if (kind == Kind::kWide)
    return launch_wide(a, plan_wide(batch, num_kv_heads, head_dim, G, rows, tokens, cap),
                       head_dim, workspace, stream);
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = need ? reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                              part_o_bytes(p, head_dim))
                   : nullptr;
  a.W = p.W;
  if (kind == Kind::kToken) return launch_token(a, p, head_dim, stream);
  const long long groups = p.W != 0 ? p.W : p.segs;
  a.per_xcd = static_cast<int>((groups + 7) / 8);
  const dim3 grid(static_cast<unsigned>(8 * a.per_xcd));
  // (a byte of K/V that one row tile alone reads is streamed past the caches)
  const bool once = rows == 0 && tokens * G <= kRows;
  if (head_dim == 128) {
    if (once)
      hipLaunchKernelGGL((gqa_chunk_rows_kernel<128, 2>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((gqa_chunk_rows_kernel<128, 0>), grid, dim3(kThreads), 0, stream, a);
  } else {
    if (once)
      hipLaunchKernelGGL((gqa_chunk_rows_kernel<64, 2>), grid, dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((gqa_chunk_rows_kernel<64, 0>), grid, dim3(kThreads), 0, stream, a);
  }
  const int rc = VOOM_LAUNCH_CHECK("paged_gqa_chunk: kernel launch");
  if (rc || p.W == 0) return rc;
  return head_dim == 128 ? launch_reduce<128, Geo<128>>(a, stream)
                         : launch_reduce<64, Geo<64>>(a, stream);
}
