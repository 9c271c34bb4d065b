// Attention of ragged chunks with up to 16 rows a kv head, a decode step's single tokens
// (gqa_chunk.hip has the formulas, chunk_rows.h the scores).
//
// What bounds it: K and V of the tokens seen, read once.
//
// A row tile is the 16 columns of v_mfma_f32_16x16x32_bf16: the (new token, head of the
// group) rows of a (sequence, kv head) up to 16 at a time.  A wavefront streams 32-token
// blocks straight into its operand registers, two blocks ahead of the one that it computes,
// without LDS or barriers (through the ring in LDS that 64 rows share, gqa_chunk_rows_kernel,
// 16 requests of up to 32,768 tokens, 32/8 heads of 128, took 197 us where this takes 154).
// Blocks behind the prefix and before the window are left out.
//
// Where segments are long their blocks lie end to end, each segment's after kLead units that
// stand for what it costs besides, and are dealt out evenly to four wavefronts a CU;
// gqa_chunk_reduce_kernel merges the cut ones.  Where they are short a workgroup's wavefronts
// share one and merge it in LDS: one launch.
#include "chunk_few.h"

#include <climits>

namespace voom {
namespace {

constexpr int kTileRows = 16;
constexpr int kAhead = 2;          // blocks in flight besides the one computed
constexpr int kSplitWaves = 4;     // wavefronts of a workgroup, split
constexpr int kSegWaves = 4;       // and of one that walks a whole segment
constexpr int kShort = 24;         // blocks of 128 dims of a segment that is not cut
// (3 units at least: 16,000 tokens of one sequence, 3 kv heads of 64: 15.5 us, with 1 22 us)
typedef Geometry<kTileRows, kBlk, 4, 3> Geo;

// A wavefront's walk over blocks of one segment.
template <int D>
struct Walk {
  const ChunkArgs& a;
  int lane, kvh, pre, gap, ctx, prefix;
  const int32_t* row;   // the sequence's table row
  int tab_base, tab;    // first page of those in the lanes, and their slots
  u32x4 qop[D / 32];
  View view;
  int lo_max, hi_min;   // what all rows of the tile see
  bool live;            // this lane's row is one
  int t_row, head;
  size_t out_row;

  __device__ __forceinline__ Walk(const ChunkArgs& args, int b, int kvh_, int tile, int pre_,
                                  int gap_, int lane_)
      : a(args), lane(lane_), kvh(kvh_), pre(pre_), gap(gap_), tab_base(-(1 << 30)), tab(0) {
    ctx = uniform(context_of(a, b));
    int base;
    const int n = uniform(new_of(a, b, base));
    prefix = uniform(prefix_of(a, b, ctx));
    row = a.table + static_cast<size_t>(b) * a.max_pages;
    const int r = tile * kTileRows + (lane & 15);
    t_row = r / a.G;
    live = t_row < n;
    head = kvh * a.G + (r - t_row * a.G);
    out_row = out_at(a, b, base, t_row, head);
    const Sight sight(a, ctx, n, prefix, t_row);
    view.ctx = ctx;
    view.pre = live ? prefix : 0;
    view.at = sight.at;
    view.lo = sight.lo;
    view.hi = live ? sight.hi : 0;
    view.biased = a.slopes != nullptr;
    view.slope = view.biased ? a.slopes[head] * 1.4426950408889634f : 0.f;
    const int t_lo = tile * kTileRows / a.G;
    int t_hi = (tile * kTileRows + kTileRows - 1) / a.G;
    t_hi = t_hi < n ? t_hi : n - 1;
    hi_min = Sight(a, ctx, n, prefix, t_lo).hi;
    lo_max = Sight(a, ctx, n, prefix, t_hi).lo;
    const uint16_t* qr =
        a.q + (live ? query_at(a, b, base, t_row, head) * D : 0) + 8 * (lane >> 4);
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
      qop[s] = live ? *reinterpret_cast<const u32x4*>(qr + 32 * s) : u32x4{};
  }

  // Block c of the segment: the context's 32-token block.
  __device__ __forceinline__ int block(int c) const { return c < pre ? c : c + gap; }

  // Block c into o; one past the end (c >= end) is read from nowhere, as zeros, so that the
  // waits in front of each block do not depend on a branch.
  __device__ __forceinline__ void load(Operands<D>& o, int c, int end) {
    const bool in = c < end;
    const int bi = block(in ? c : end - 1);
    const int sub_shift = a.pt_shift - 5;
    const int page = bi >> sub_shift;
    if (page < tab_base || page >= tab_base + kWave) {
      tab_base = page;
      const int p = page + lane;
      tab = p < a.max_pages ? row[p] : 0;
      wait_vmem_all();  // here, not at the readlane of every block
    }
    int slot = __builtin_amdgcn_readlane(tab, page - tab_base);
    if (static_cast<unsigned>(slot) >= static_cast<unsigned>(a.num_slots)) slot = 0;
    const size_t at = (((static_cast<size_t>(slot) * a.NKV + kvh) << sub_shift) +
                       (bi - (page << sub_shift))) * (kBlk * D);
    const int bytes = in ? kBlk * D * 2 : 0;
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(a.k_pool + at), static_cast<short>(0), bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(a.v_pool + at), static_cast<short>(0), bytes, 0x00020000);
    const int i16 = lane & 15, g = lane >> 4;
    const int k_lane = ((8 * (i16 >> 2) + (i16 & 3)) * D + 8 * g) * 2;
    const int v_lane = (i16 * kBlk + 8 * g) * 2;
    // (every byte is read once: streamed past the caches)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
        o.k[s][t] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane + (4 * t * D + 32 * s) * 2,
                                                          0, 2);
    }
#pragma unroll
    for (int n = 0; n < D / 16; ++n)
      o.v[n] = __builtin_amdgcn_raw_buffer_load_b128(vr, v_lane + n * (16 * kBlk * 2), 0, 2);
  }

  __device__ __forceinline__ void compute(const Operands<D>& o, int c, State<D, 1>& st) {
    const int first = block(c) * kBlk;
    const int pos = first + 8 * (lane >> 4);
    f32x4 sc[1][2];
    u32x4 p[1];
    const u32x4(&q)[1][D / 32] = reinterpret_cast<const u32x4(&)[1][D / 32]>(qop);
    scores_of<D, 1>(o, q, sc);
    score(sc, a, view, pos);
    if ((first >= lo_max && first + kBlk <= hi_min) || first + kBlk <= prefix) {
      weights_of<D>(sc, st, p);
      products<D, 1>(o, p, st);
      return;
    }
    const uint32_t seen = view.seen(pos);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sc[0][e >> 2][e & 3] = (seen >> e & 1) != 0 ? sc[0][e >> 2][e & 3] : -INFINITY;
    weights_of<D>(sc, st, p);
    masked_products<D, 1>([&](int n) { return o.v[n]; }, p, st, ctx - pos,
                          [&](int) { return seen; });
  }

  // Blocks [begin, end), at least one.
  __device__ __forceinline__ void run(int begin, int end, State<D, 1>& st) {
    Operands<D> ring[kAhead + 1];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) load(ring[j], begin + j, end);
    for (int c = begin; c < end; c += kAhead + 1) {
#pragma unroll
      for (int j = 0; j <= kAhead; ++j) {
        load(ring[(j + kAhead) % (kAhead + 1)], c + j + kAhead, end);
        if (c + j < end) compute(ring[j], c + j, st);
      }
    }
  }
};

template <int D>
__device__ __forceinline__ void clear(State<D, 1>& st) {
  // never -inf: keys of score -inf then weigh 0 also where nothing came before
  st.m[0] = -FLT_MAX;
  st.l[0] = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) st.acc[0][i] = f32x4{};
}

template <int D>
__global__ __launch_bounds__(kSplitWaves * kWave, 1) void gqa_chunk_split_kernel(ChunkArgs a) {
  constexpr int kLead = Geo::kLead;
  const int lane = threadIdx.x & (kWave - 1);
  const int w = static_cast<int>(blockIdx.x) * kSplitWaves + uniform(threadIdx.x / kWave);
  int x0;
  const Units<Geo> first = scan_units<Geo>(a, 0, lane, x0);
  int U = __builtin_amdgcn_readlane(x0, kWave - 1);
  for (int base = kWave; base < a.B; base += kWave) {
    int x;
    scan_units<Geo>(a, base, lane, x);
    U += __builtin_amdgcn_readlane(x, kWave - 1);
  }
  const Split split = split_of<Geo>(U, a.W);
  if (w >= split.We || U == 0) return;
  int u0 = split.begin(w);
  const int u1 = split.begin(w + 1);
  int b = 0, kvh, tile, chunks = 0, tiles = 1, pre = 0, gap = 0, begin = 0;
  for (int base = 0;; base += kWave) {  // the sequence that holds unit u0
    if (base >= a.B) return;
    int x = x0;
    Units<Geo> units = first;
    if (base != 0) units = scan_units<Geo>(a, base, lane, x);
    const int here = __builtin_amdgcn_readlane(x, kWave - 1);
    if (u0 < begin + here) {
      const int k = __popcll(__builtin_amdgcn_ballot_w64(begin + x <= u0));
      b = base + k;
      chunks = __builtin_amdgcn_readlane(units.chunks, k);
      tiles = __builtin_amdgcn_readlane(units.tiles, k);
      pre = __builtin_amdgcn_readlane(units.pre, k);
      gap = __builtin_amdgcn_readlane(units.gap, k);
      begin += __builtin_amdgcn_readlane(x, k) - (chunks + kLead) * tiles * a.NKV;
      break;
    }
    begin += here;
  }
  {
    const int s = (u0 - begin) / (chunks + kLead);
    kvh = s / tiles;
    tile = s - kvh * tiles;
    begin += s * (chunks + kLead);
  }
  while (true) {
    const int at = begin + kLead;  // the segment's first block
    if (u1 <= at) return;
    const int c0 = u0 > at ? u0 - at : 0;
    const int c1 = (u1 < at + chunks ? u1 : at + chunks) - at;
    Walk<D> walk(a, b, kvh, tile, pre, gap, lane);
    State<D, 1> st;
    clear<D>(st);
    walk.run(c0, c1, st);
    const float lt = wave_sum_across_groups(st.l[0]);
    const int i16 = lane & 15, g = lane >> 4;
    if (c0 == 0 && c1 == chunks) {
      const bool empty = lt == 0.f;
      const float inv = 1.f / lt;
      if (walk.live) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const f32x4 o = st.acc[0][i];
          *reinterpret_cast<u32x2*>(a.out + walk.out_row * D + 16 * i + 4 * g) =
              empty ? u32x2{0u, 0u}
                    : u32x2{pack_bf16x2(o[0] * inv, o[1] * inv),
                            pack_bf16x2(o[2] * inv, o[3] * inv)};
        }
        if (g == 0 && a.lse != nullptr)
          a.lse[walk.out_row] =
              empty ? -INFINITY : (st.m[0] + __log2f(lt)) * 0.6931471805599453f;
      }
    } else if (walk.live) {
      const size_t p = (2 * static_cast<size_t>(w) + (c0 == 0 ? 1 : 0)) * kTileRows + i16;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<f32x4*>(a.part_o + p * D + 16 * i + 4 * g) = st.acc[0][i];
      if (g == 0) *reinterpret_cast<float2*>(a.part_ml + p * 2) = {st.m[0], lt};
    }
    begin += kLead + chunks;
    u0 = u1 < begin ? u1 : begin;
    if (u0 >= u1) return;
    if (++tile == tiles) {
      tile = 0;
      if (++kvh == a.NKV) {
        kvh = 0;
        do {
          const Units<Geo> units(a, ++b);
          chunks = uniform(units.chunks);
          tiles = uniform(units.tiles);
          pre = uniform(units.pre);
          gap = uniform(units.gap);
        } while (b < a.B - 1 && chunks == 0);
      }
    }
  }
}

// A workgroup per segment.
template <int D>
__global__ __launch_bounds__(kSegWaves * kWave) void gqa_chunk_segment_kernel(ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) float part_o[kSegWaves][kTileRows][D + 4];
  __shared__ float part_m[kSegWaves][kTileRows], part_l[kSegWaves][kTileRows];
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = uniform(threadIdx.x / kWave);
  const int w = static_cast<int>(blockIdx.x);
  int b = 0, tiles = 1, chunks = 0, pre = 0, gap = 0, begin = 0;
  for (int base = 0;; base += kWave) {  // the sequence that holds segment w
    if (base >= a.B) return;
    int x;
    const Units<Geo> units = scan_units<Geo>(a, base, lane, x);
    const int here = __builtin_amdgcn_readlane(x, kWave - 1);
    if (w < begin + here) {
      const int k = __popcll(__builtin_amdgcn_ballot_w64(begin + x <= w));
      b = base + k;
      chunks = __builtin_amdgcn_readlane(units.chunks, k);
      tiles = __builtin_amdgcn_readlane(units.tiles, k);
      pre = __builtin_amdgcn_readlane(units.pre, k);
      gap = __builtin_amdgcn_readlane(units.gap, k);
      begin += __builtin_amdgcn_readlane(x, k) - tiles * a.NKV;
      break;
    }
    begin += here;
  }
  const int kvh = (w - begin) / tiles;
  const int tile = w - begin - kvh * tiles;
  Walk<D> walk(a, b, kvh, tile, pre, gap, lane);
  State<D, 1> st;
  clear<D>(st);
  const int c0 = wv * chunks / kSegWaves, c1 = (wv + 1) * chunks / kSegWaves;
  if (c0 < c1 && __builtin_amdgcn_ballot_w64(walk.live) != 0) walk.run(c0, c1, st);
  const int i16 = lane & 15, g = lane >> 4;
  const float lt = wave_sum_across_groups(st.l[0]);
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    *reinterpret_cast<f32x4*>(&part_o[wv][i16][16 * i + 4 * g]) = st.acc[0][i];
  if (g == 0) {
    part_m[wv][i16] = st.m[0];
    part_l[wv][i16] = lt;
  }
  __syncthreads();
  // a row at a time to a wavefront, its dims to the lanes
  int base;
  const int n = uniform(new_of(a, b, base));
  constexpr int DPL = D / kWave;
  for (int r = wv; r < kTileRows; r += kSegWaves) {
    const int row = tile * kTileRows + r;
    const int t = row / a.G;
    if (a.starts != nullptr ? t >= n : t >= a.T) return;
    float M = part_m[0][r];
#pragma unroll
    for (int i = 1; i < kSegWaves; ++i) M = fmaxf(M, part_m[i][r]);
    float L = 0.f, o[DPL] = {};
#pragma unroll
    for (int i = 0; i < kSegWaves; ++i) {
      const float f = fast_exp2(part_m[i][r] - M);
      L += part_l[i][r] * f;
#pragma unroll
      for (int d = 0; d < DPL; ++d) o[d] += part_o[i][r][lane * DPL + d] * f;
    }
    const bool empty = t >= n || L == 0.f;
    const float inv = 1.f / L;
    const size_t at = out_at(a, b, base, t, kvh * a.G + (row - t * a.G));
#pragma unroll
    for (int d = 0; d < DPL; ++d)
      a.out[at * D + lane * DPL + d] = empty ? 0 : f2bf(o[d] * inv);
    if (lane == 0 && a.lse != nullptr)
      a.lse[at] = empty ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
  }
}

}  // namespace

FewPlan plan_token(int B, int NKV, int D, int G, int N, int T, long long tokens, int window) {
  FewPlan p;
  const long long tiles = N > 0 ? static_cast<long long>(N) * G / kTileRows + (B < N ? B : N)
                                : static_cast<long long>(B) * ((T * G + kTileRows - 1) / kTileRows);
  p.segs = tiles * NKV;
  long long blocks = (tokens + kBlk - 1) / kBlk;
  const long long seen = (static_cast<long long>(window) + kTileRows / G) / kBlk + 2;
  if (seen < blocks) blocks = seen;
  // One launch where contexts are short, the longer the better their segments fill the card
  // (8 kv heads, without and with the split: 8 segments of 128 dims and 500 tokens 12.1 and
  // 13.7 us, of 1,000 16.6 and 14.0; 256 of them 24 and 27.6, of 2,000 44 and 49; 3 segments
  // of 64 dims and 1,000 tokens 10.9 and 13.9, of 2,000 17.5 and 14.5).
  const int cus = device_cu_count();
  const long long full = (p.segs + cus - 1) / cus * cus;
  const int most = 16 * p.segs >= 15 * full ? 64 : kShort * (128 / D);
  p.W = blocks <= most ? 0 : kSplitWaves * cus;
  p.rows = kTileRows;
  return p;
}

int launch_token(const ChunkArgs& a, const FewPlan& p, int D, hipStream_t stream) {
  if (p.W == 0) {
    const dim3 grid(static_cast<unsigned>(p.segs)), block(kSegWaves * kWave);
    if (D == 128) hipLaunchKernelGGL(gqa_chunk_segment_kernel<128>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(gqa_chunk_segment_kernel<64>, grid, block, 0, stream, a);
    return VOOM_LAUNCH_CHECK("paged_gqa_chunk: segment launch");
  }
  const dim3 grid(static_cast<unsigned>(p.W / kSplitWaves)), block(kSplitWaves * kWave);
  if (D == 128) hipLaunchKernelGGL(gqa_chunk_split_kernel<128>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(gqa_chunk_split_kernel<64>, grid, block, 0, stream, a);
  const int rc = VOOM_LAUNCH_CHECK("paged_gqa_chunk: split launch");
  if (rc) return rc;
  return D == 128 ? launch_reduce<128, Geo>(a, stream) : launch_reduce<64, Geo>(a, stream);
}

}  // namespace voom
