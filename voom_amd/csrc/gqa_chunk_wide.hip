// Attention of ragged chunks with many rows (gqa_chunk.hip has the formulas, chunk_rows.h
// the scores): long parts of prompts, alone or beside single tokens.
//
// What bounds it: matrix work, 4 NQ D flops per (new token, token seen), beside an
// exponential per score and, with a cap, a polynomial of it.  Neither unit is busy all of the
// time: tiles wait for their stage, and workers for the longest one.
//
// A row tile is 128 rows (new token, head of the group) of a (sequence, kv head): four
// wavefronts of 32 rows, which share 64-key tiles of K and V^T in LDS, loaded straight into
// one of two buffers while the other is computed.  Per tile and wavefront, on
// v_mfma_f32_32x32x16_bf16 with the rows in the N dimension:
//   scores^T[64 keys][32 rows] = K . Q^T,  out^T[D dims][32 rows] += V^T . P^T
// The key rows of the score operand are permuted (key_of_row), so that a lane's scores are
// the keys that its P^T operand needs.  The scores run a tile ahead: those of tile t + 1 are
// formed while the exponentials of tile t are taken, and become logits (cap, slopes,
// maximum) during P.V of tile t.  Tiles that every row of the wavefront sees whole take that
// loop, those at the window's edge and the diagonal one with masks, two at a time.
//
// gqa_chunk_plan_kernel lists the row tiles of all sequences, from their lengths on the
// device, and cuts long ones over keys, so that the workgroups are done at about the same time;
// the pieces leave (m, l, o) in fp32 and gqa_chunk_join_kernel merges them.
//
// The last 2,011 of 6,007 tokens, 32/8 heads of 128, capped: 192-196 us a call, one behind
// another, 850 TFLOP/s, of which the plan 6 and the join 5 (row tiles of 64 through the ring of
// gqa_chunk.hip: 663 us).  The plan's 504 uncut pieces leave 17 % of the workers' time idle.
#include "chunk_rows.h"

#include <cfloat>
#include <climits>
#include <type_traits>

namespace voom {
namespace {

constexpr int kBlk = 32;        // tokens of a K/V block in the pool
constexpr int kKeys = 64;       // keys per tile
constexpr int kRows = 32;       // rows of a wavefront
constexpr int NW = 4;           // wavefronts of a workgroup
constexpr int kTileRows = NW * kRows;
constexpr int kAhead = 4;       // operand reads ahead of the MFMAs
constexpr int kMinPiece = 8;    // tiles of a piece at least
constexpr float kSlack = 8.f;   // the reference maxima stay that far behind, in log2 units

// (a lambda that is called would have its captures in scratch memory)
#define VOOM_INLINE __attribute__((always_inline))

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

struct WideArgs {
  ChunkArgs c;
  int32_t* head;   // row tiles of a kv head that are cut
  int4* pieces;    // {sequence, row tile, first and last + 1 of its key tiles}, and its
                   // sequence's {context, new tokens, prefix} and where the piece leaves its
                   // state, -1: it is the whole row tile
  int4* cuts;      // {sequence, row tile, pieces, first slot}, {new tokens, first row}
  int32_t* lengths;  // key tiles of the row tiles
  WidePlan p;
};

// The key tiles that the rows of a row tile see: those of the prefix, and from `gap` tiles
// further on.
struct KeyTiles {
  int pre, gap, count;
  __device__ __forceinline__ KeyTiles(const ChunkArgs& a, int ctx, int n, int prefix, int rt) {
    const int t0 = rt * kTileRows / a.G;
    if (t0 >= n || ctx == 0) {
      pre = gap = count = 0;
      return;
    }
    const int t1 = (rt * kTileRows + kTileRows - 1) / a.G;
    const Sight first(a, ctx, n, prefix, t0);
    const Sight last(a, ctx, n, prefix, t1 < n ? t1 : n - 1);
    pre = (prefix + kKeys - 1) / kKeys;
    gap = first.lo / kKeys - pre;
    gap = gap < 0 ? 0 : gap;
    count = (last.hi + kKeys - 1) / kKeys - gap;
    count = count < 0 ? 0 : count;
  }
  __device__ __forceinline__ int tile(int c) const { return c < pre ? c : c + gap; }
};

// Cuts the row tiles of all sequences into pieces.  A piece has at most `most` key tiles; of
// some candidates the one is taken with which the workers are done first.  Each piece costs
// kLead key tiles besides its own, kCutLead where it also leaves its state to be merged.  Where
// all pieces run at once, a CU's two workers are a long and a short one; else a worker has its
// share, and at the end half a piece more or less than others.  Pieces are listed in falling
// length.
constexpr int kPlanThreads = 256;
constexpr int kHeld = 2048;      // row tiles whose lengths are held in LDS
constexpr int kClasses = 64;     // of lengths
constexpr int kTries = 8;
constexpr float kLead = 3.f, kCutLead = 9.f;
constexpr float kCaps[kTries] = {0.f, 2.f, 1.5f, 1.2f, 1.f, 0.8f, 0.6f, 0.4f};  // of a share

__global__ __launch_bounds__(kPlanThreads) void gqa_chunk_plan_kernel(WideArgs w) {
  constexpr int kPlanWaves = kPlanThreads / kWave;
  const ChunkArgs& a = w.c;
  __shared__ int first[kMaxChunkBatch + 1];  // row tiles before each sequence
  __shared__ int4 seqs[kMaxChunkBatch];      // context, new tokens, prefix, first row
  __shared__ int held[kHeld];
  __shared__ int sums[kPlanWaves];
  __shared__ float alls[kPlanWaves], tops[kPlanWaves];
  __shared__ int tried[kTries], classes[kClasses], slots, cuts;
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & (kWave - 1);
  const int wv = uniform(tid / kWave);
  if (tid < kClasses) classes[tid] = 0;
  if (tid < kTries) tried[tid] = 0;
  if (tid == 0) {
    slots = cuts = 0;
    first[0] = 0;
  }
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int tiles = 0;
    if (b < a.B) {
      int base;
      const int ctx = context_of(a, b), n = new_of(a, b, base);
      seqs[b] = {ctx, n, prefix_of(a, b, ctx), base};
      tiles = ((a.starts != nullptr ? n : a.T) * a.G + kTileRows - 1) / kTileRows;
    }
    const int x = wave_inclusive_scan(tiles, lane);
    if (lane == kWave - 1) sums[wv] = x;
    __syncthreads();
    int here = 0, total = 0;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) {
      here += i < wv ? sums[i] : 0;
      total += sums[i];
    }
    if (b < a.B) first[b + 1] = before + here + x;
    before += total;
    __syncthreads();
  }
  const int entries = before < w.p.entries ? before : w.p.entries;  // (starts that overlap)
  // row tile e: its sequence, its place there (the last, which sees most, first), key tiles
  auto place = [&](int e, int& b, int& rt) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= e) lo = mid;
      else hi = mid;
    }
    b = lo;
    rt = first[lo + 1] - 1 - e;
  };
  auto length = [&](int e) -> int& { return e < kHeld ? held[e] : w.lengths[e]; };
  // (sums in fp32: they weigh candidates, and bound nothing by less than a tile)
  float mine = 0.f, top = 0.f;
  for (int e = tid; e < entries; e += kPlanThreads) {
    int b, rt;
    place(e, b, rt);
    const int n = KeyTiles(a, seqs[b].x, seqs[b].y, seqs[b].z, rt).count;
    length(e) = n;  // (read again by this thread alone)
    mine += static_cast<float>(n);
    top = fmaxf(top, static_cast<float>(n));
  }
  mine = wave_sum_uniform(mine);
  top = wave_max_uniform(top);
  if (lane == 0) {
    alls[wv] = mine;
    tops[wv] = top;
  }
  __syncthreads();
  mine = (alls[0] + alls[1]) + (alls[2] + alls[3]);
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float share = mine * a.NKV / w.p.workers;  // of a worker
  // a candidate's key tiles of a piece; no piece so short that the workspace could not hold
  // all of them
  auto limit_of = [&](float cap) {
    const float least = floorf(share * kCaps[kTries - 1]) + 1.f;
    return fmaxf(fminf(cap == 0.f ? top : floorf(share * cap) + 1.f, top),
                 fmaxf(least, static_cast<float>(kMinPiece)));
  };
  // pieces of n key tiles, `most` in each (in fp32: one more now and then is no matter)
  auto parts_of = [&](int n, float most) {
    const float x = static_cast<float>(n);
    return x > most ? static_cast<int>(ceilf(x * __builtin_amdgcn_rcpf(most))) : 1;
  };
  {
    int parts[kTries] = {};
    for (int e = tid; e < entries; e += kPlanThreads) {
      const int n = length(e);
#pragma unroll
      for (int i = 0; i < kTries; ++i) parts[i] += n > 0 ? parts_of(n, limit_of(kCaps[i])) : 0;
    }
#pragma unroll
    for (int i = 0; i < kTries; ++i) {
      const int n = __builtin_amdgcn_readlane(wave_inclusive_scan(parts[i], lane), kWave - 1);
      if (lane == 0) atomicAdd(&tried[i], n);
    }
  }
  __syncthreads();
  float most;
  {  // a candidate a lane
    float cap = 0.f;
#pragma unroll
    for (int i = 1; i < kTries; ++i) cap = lane % kTries == i ? kCaps[i] : cap;
    most = limit_of(cap);
    const float pieces = static_cast<float>(tried[lane % kTries]) * a.NKV;
    const float lead = tried[lane % kTries] > tried[0] ? kCutLead : kLead;
    const float part = fminf(top, most);
    const float mean = mine * a.NKV / pieces;  // key tiles of a piece
    const float rounds = pieces / w.p.workers;
    float cost = rounds <= 1.f ? 0.5f * (part + share) + lead
                               : fmaxf(part + lead, share + lead * rounds + 0.5f * mean);
    float best = cost;
#pragma unroll
    for (int k = 1; k < kTries; k <<= 1) best = fminf(best, __shfl_xor(best, k));
    const uint64_t hit = __builtin_amdgcn_ballot_w64(cost == best);
    most = __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, most),
                                         hit != 0 ? __builtin_ctzll(hit) : 0));
  }
  const float step = (kClasses - 1) / (fminf(top, most) + 1.f);
  // the class of a piece's length, the longest first
  auto class_of = [&](int n, int parts) {
    const int c = static_cast<int>(n * step / parts);
    return kClasses - 1 - (c < kClasses ? c : kClasses - 1);
  };
  for (int e = tid; e < entries; e += kPlanThreads) {
    const int n = length(e);
    const int parts = parts_of(n, most);
    atomicAdd(&classes[class_of(n, parts)], parts);
  }
  __syncthreads();
  if (wv == 0) {
    const int n = classes[lane];
    const int x = wave_inclusive_scan(n, lane);
    classes[lane] = x - n;
    if (lane == kWave - 1) sums[0] = x;
  }
  __syncthreads();
  const int listed = sums[0] < w.p.pieces ? sums[0] : w.p.pieces;
  // Of the pieces that run from the start, two a CU, the second half is dealt the other way
  // round: a CU then has a long one and a short one.
  const int half = w.p.workers / 2 / a.NKV;
  auto dealt = [&](int p, int n) {
    const int end = n < 2 * half ? n : 2 * half;
    return p < half || p >= end ? p : half + end - 1 - p;
  };
  for (int e = tid; e < entries; e += kPlanThreads) {
    const int n = length(e);
    const int parts = parts_of(n, most);
    int b, rt, s = -1;
    place(e, b, rt);
    const int4 seq = seqs[b];
    if (parts > 1) {
      s = atomicAdd(&slots, parts);
      const int k = atomicAdd(&cuts, 1);
      if (k < w.p.cuts) {
        w.cuts[2 * k] = {b, rt, parts, s};
        w.cuts[2 * k + 1] = {seq.y, seq.w, 0, 0};
      }
    }
    int p = atomicAdd(&classes[class_of(n, parts)], parts);
    const int each = n / parts, more = n - each * parts;  // `more` of them one tile longer
    int from = 0;
    for (int i = 0; i < parts && p < w.p.pieces; ++i, ++p) {
      const int to = from + each + (i < more ? 1 : 0);
      const int at = dealt(p, listed);
      w.pieces[2 * at] = {b, rt, from, to};
      w.pieces[2 * at + 1] = {seq.x, seq.y, seq.z, s < 0 || s + i >= w.p.slots ? -1 : s + i};
      from = to;
    }
  }
  for (int p = listed + tid; p < w.p.pieces; p += kPlanThreads)
    w.pieces[2 * p] = {-1, 0, 0, 0};
  __syncthreads();
  if (tid == 0) w.head[0] = cuts < w.p.cuts ? cuts : w.p.cuts;
}

// Key (0..31 of a block) that row r of the score tile holds: lane half h then
// has keys 8h..8h+7 in its first eight accumulators and 16+8h.. in the others.
__device__ __forceinline__ int key_of_row(int r) {
  return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3);
}
// Key of accumulator i of block j, less 8 times the lane's half.
constexpr int key_of(int j, int i) { return 32 * j + 16 * (i >> 3) + (i & 7); }

// Chunk c (16 bytes) of K row r sits at c ^ k_swizzle(r): 16 consecutive keys
// then read one chunk from 16 different 16-byte columns.
template <int D>
__device__ __forceinline__ int k_swizzle(int r) {
  return D == 128 ? (r & 15) : ((r >> 1) & 7);
}

// CAP: scores capped by a tanh; BIAS: lowered with the distance (also by slopes of 0, for
// scales that are not positive: without either the raw scores' maximum stands for theirs).
template <int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(NW * kWave) __attribute__((amdgpu_waves_per_eu(2, 2)))
void gqa_chunk_tiles_kernel(WideArgs wa) {
  constexpr bool kMod = CAP || BIAS;           // scores become logits before the maximum
  constexpr int kBlkElems = kBlk * D;          // elements of one K or V block
  constexpr int kPieces = kBlkElems / 512;     // 1 KiB loads per block
  constexpr int kLoads = 4 * kPieces / NW;     // loads per wavefront and tile
  constexpr int kCpr = D / 8;                  // 16-byte chunks of a K row
  constexpr int KS = D / 16;                   // k-steps of the scores
  constexpr int DT = D / 32;                   // dim tiles of out^T
  // masks of __builtin_amdgcn_sched_group_barrier
  constexpr int kValu = 0x002, kMfma = 0x008, kVmemRead = 0x020, kDsRead = 0x100, kTrans = 0x400;
  static_assert(kLoads * NW == 4 * kPieces, "loads split evenly over the wavefronts");
  // K block 0, K block 1, V^T block 0, V^T block 1.  Two distinct objects, so
  // that reads of one provably miss the other's pending direct-to-LDS loads.
  __shared__ __attribute__((aligned(1024))) uint16_t tile_a[4 * kBlkElems];
  __shared__ __attribute__((aligned(1024))) uint16_t tile_b[4 * kBlkElems];
  __shared__ int again;
  const ChunkArgs& a = wa.c;

  // A piece for all kv heads in turn: an XCD takes every eighth, so that the heads of its
  // pieces, and with them K and V in its L2, are few.
  const int in_head = static_cast<int>(blockIdx.x) / a.NKV;
  const int kvh = static_cast<int>(blockIdx.x) - in_head * a.NKV;
  const int4 piece = wa.pieces[2 * in_head], seq = wa.pieces[2 * in_head + 1];
  const int b = uniform(piece.x);
  if (b < 0) return;
  const int rt = uniform(piece.y);
  const int c_lo = uniform(piece.z);
  const int c_hi = uniform(piece.w);
  const int ctx = uniform(seq.x);
  const int n = uniform(seq.y);
  const int prefix = uniform(seq.z);
  const int slot = uniform(seq.w);
  const int base = a.starts != nullptr ? clamped(uniform(a.starts[b]), a.N) : 0;
  const KeyTiles keys(a, ctx, n, prefix, rt);
  const int R = n * a.G;  // rows of the sequence

  const int lane = threadIdx.x & (kWave - 1);
  const int w = uniform(threadIdx.x / kWave) & (NW - 1);
  const int l32 = lane & 31;
  const int lh = lane >> 5;

  // This lane's row (rows past the sequence's repeat its last one and are not stored), what
  // it sees, and what all and any of the wavefront see.
  const int row = rt * kTileRows + w * kRows + l32;
  const int rc = row < R ? row : (R > 0 ? R - 1 : 0);
  const int tok = rc / a.G;
  const int head = kvh * a.G + (rc - tok * a.G);
  const Sight sight(a, ctx, n, prefix, tok);
  const int lo = sight.lo, hi = sight.hi;
  // (a wavefront behind the sequence's last row sees nothing: it only loads)
  const bool has_rows = rt * kTileRows + w * kRows < R;
  const int lo_min = uniform(lo), hi_max = has_rows ? __builtin_amdgcn_readlane(hi, 31) : 0;
  const int lo_max = __builtin_amdgcn_readlane(lo, 31);
  // (distances of later tokens, in a prefix, have the other sign: not in the loop without masks)
  const int hi_all = uniform(hi), at_min = uniform(sight.at);
  const int hi_min = BIAS && at_min + 1 < hi_all ? (at_min + 1 > 0 ? at_min + 1 : 0) : hi_all;
  auto any_sees = [&](int t) VOOM_INLINE {
    return t * kKeys < hi_max && ((t + 1) * kKeys > lo_min || t * kKeys < prefix);
  };

  // Q^T operand: lane (row l32, half lh) holds q[16 s + 8 lh .. + 8]
  u32x4 qop[KS];
  auto load_q = [&]() VOOM_INLINE {
    const uint16_t* qh = a.q + query_at(a, b, base, tok, head) * D + 8 * lh;
#pragma unroll
    for (int s = 0; s < KS; ++s) qop[s] = *reinterpret_cast<const u32x4*>(qh + 16 * s);
  };

  // Pool blocks (K and V alike, in units of 32 tokens of one kv head) of the
  // sequence's 32-token blocks win .. win + 63, one per lane; blocks past the
  // last token repeat it (their keys are masked).
  const int32_t* trow = a.table + static_cast<size_t>(b) * a.max_pages;
  const int sub_shift = a.pt_shift - 5;
  const int last_blk = ctx > 0 ? (ctx - 1) / kBlk : 0;
  int win = -kWave;
  int blocks = 0;
  auto fill_window = [&](int bi) VOOM_INLINE {
    win = bi;
    const int mine = bi + lane < last_blk ? bi + lane : last_blk;
    const int page = mine >> sub_shift;
    int s = trow[page];
    if (static_cast<unsigned>(s) >= static_cast<unsigned>(a.num_slots)) s = 0;
    blocks = ((s * a.NKV + kvh) << sub_shift) + (mine - (page << sub_shift));
    wait_vmem_all();  // here, not at the readlanes below on every tile
  };
  // Stage c holds K of key tile c + 1 (the scores run one tile ahead of P.V) and
  // V^T of tile c.  Its pieces of 1 KiB, 4 * kPieces of them, go piece p to
  // wavefront p % NW.  stage_blocks looks the pool blocks up (V's are K's of the
  // stage before), load_piece issues load i of this wavefront.
  int kblk0 = 0, kblk1 = 0, vblk0 = 0, vblk1 = 0;
  auto stage_blocks = [&](int c) VOOM_INLINE {
    const int bi = 2 * keys.tile(c + 1);
    if (bi >= win + kWave) fill_window(bi);  // bi is even: so is the window's start
    vblk0 = kblk0;
    vblk1 = kblk1;
    kblk0 = __builtin_amdgcn_readlane(blocks, bi - win);
    kblk1 = __builtin_amdgcn_readlane(blocks, bi - win + 1);
  };
  auto load_piece = [&](int i, uint16_t* dst) VOOM_INLINE {
    const int p = w + NW * i;
    const int blk = p / kPieces;
    const int sub = p % kPieces;
    const bool is_v = blk >= 2;
    const int j = blk & 1;
    // (sums, not a choice between variables, which would become one of addresses)
    const unsigned src = uniform((is_v ? vblk0 + 0 : kblk0 + 0) * (1 - j) +
                                 (is_v ? vblk1 + 0 : kblk1 + 0) * j);
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>((is_v ? a.v_pool : a.k_pool) + static_cast<size_t>(src) * kBlkElems),
        static_cast<short>(0), kBlkElems * 2, 0x00020000);
    const int krow = sub * (kWave / kCpr) + lane / kCpr;
    const int ksrc = krow * (D * 2) + 16 * ((lane % kCpr) ^ k_swizzle<D>(krow));
    const int vrow = sub * 16 + (lane >> 2);
    const int vsrc = vrow * (kBlk * 2) + 16 * ((lane & 3) ^ ((lane >> 4) & 3));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(dst + p * 512), 16, is_v ? vsrc : ksrc,
                                             0, 0, 0);
  };
  auto load_stage = [&](int c, uint16_t* dst) VOOM_INLINE {
    stage_blocks(c);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_piece(i, dst);
  };

  // Per-lane LDS byte addresses of the operands.  K: row key_of_row(l32),
  // chunk 2 s + lh.  V^T: dim row 32 dt + l32, chunk 2 ks + lh of its block.
  const int key = key_of_row(l32);
  const int k_lane = key * (D * 2) + 16 * (lh ^ k_swizzle<D>(key));
  int v_lane[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
    v_lane[ks] = l32 * (kBlk * 2) + 16 * ((2 * ks + lh) ^ ((l32 >> 2) & 3));

  f32x16 acc[DT];
  // Reference of the exponentials, log2 units, the same in both halves, 0 until a key of
  // any weight is seen; it is raised where a score is more than `above` ahead of it.
  float m, above;
  float l;              // over this lane's keys

  // Scores of a tile (accumulator i of block j: key key_of(j, i) + 8 lh): raw, or with kMod
  // as logits in log2 units less m.
  typedef f32x16 Scores[2];
  const float slope = BIAS && a.slopes != nullptr ? a.slopes[head] * 1.4426950408889634f : 0.f;
  // cap tanh(s cap_k) = s (q0 + q1 s^2 + q2 s^4 + q3 s^6) where |s cap_k| <= kNear
  const float k2 = a.cap_k * a.cap_k;
  const float q0 = a.scale * kTanh[0], q1 = a.scale * kTanh[1] * k2;
  const float q2 = a.scale * kTanh[2] * k2 * k2, q3 = a.scale * kTanh[3] * k2 * k2 * k2;
  const float far = CAP ? kNear / fabsf(a.cap_k) : 0.f;  // (a scale of 0: infinite)
  // The polynomial's coefficients for a tile; far scores are capped before it, and it is
  // then the identity.
  struct Poly {
    float q0, q1, q2, q3;
  };
  const Poly near{q0, q1, q2, q3};
  auto logit = [&](float s, const Poly& q, float add) VOOM_INLINE {
    if constexpr (CAP) {
      const float t = s * s;
      float p = __builtin_fmaf(t, q.q3, q.q2);
      p = __builtin_fmaf(t, p, q.q1);
      p = __builtin_fmaf(t, p, q.q0);
      return __builtin_fmaf(s, p, add);
    }
    return __builtin_fmaf(s, a.scale, add);
  };
  auto raw_far = [&](const Scores& sc) VOOM_INLINE {  // whether a score of the wavefront is far
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(fmaxf(mx, fabsf(sc[0][i])), fabsf(sc[1][i]));
    return __builtin_amdgcn_ballot_w64(mx > far) != 0;
  };
  auto cap_far = [&](Scores& sc) VOOM_INLINE {
    if (!CAP || !raw_far(sc)) return near;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float y = capped_far(sc[j][i] * a.cap_k, a.cap);
        asm volatile("" : "+v"(y));  // (a choice of values, not a branch around the exponential)
        sc[j][i] = fabsf(sc[j][i]) > far ? y : logit(sc[j][i], near, 0.f);
        __builtin_amdgcn_sched_barrier(0);  // a few values in registers at a time
      }
    }
    return Poly{1.f, 0.f, 0.f, 0.f};
  };
  // Logits of tile t, -inf where this lane's row does not see the key.
  auto mask_scores = [&](int t, Scores& sc) VOOM_INLINE {
    const int k0 = t * kKeys + 8 * lh;
    const int rel_lo = lo - k0, rel_hi = hi - k0, rel_pre = prefix - k0;
    if constexpr (kMod) {
      auto add = [&](int j, int i) VOOM_INLINE {
        if constexpr (!BIAS) return -m;
        const int d = sight.at - k0 - key_of(j, i);
        return __builtin_fmaf(-slope, static_cast<float>(d < 0 ? -d : d), -m);
      };
      const Poly poly = cap_far(sc);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sc[j][i] = logit(sc[j][i], poly, add(j, i));
          if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (t * kKeys >= lo_max && t * kKeys >= prefix) {  // the diagonal alone
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[j][i] = key_of(j, i) < rel_hi ? sc[j][i] : -INFINITY;
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int k = key_of(j, i);
        sc[j][i] = (k >= rel_lo && k < rel_hi) || k < rel_pre ? sc[j][i] : -INFINITY;
      }
    }
  };
  auto max_of = [&](const Scores& sc) VOOM_INLINE {
    float mx = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(fmaxf(mx, sc[0][i]), sc[1][i]);
    return mx;
  };
  // Raises the references to a tile's maxima (mx: this lane's) before its P is formed, if
  // one is more than `above` behind: weights of up to 2^kSlack lose nothing.
  auto raise = [&](float mx, Scores& sc) VOOM_INLINE {
    const float ahead = kMod ? mx : __builtin_fmaf(mx, a.scale, -m);
    if (__builtin_amdgcn_ballot_w64(ahead > above) == 0) return;
    const float both = fmaxf(ahead, __shfl_xor(ahead, 32));
    const float up = both > above ? both : 0.f;
    float alpha = above > 0.f ? fast_exp2(-up) : 1.f;  // (nothing to rescale before the first)
    asm volatile("" : "+v"(alpha));  // keeps the rescaling inside the branch
    above = both > above ? kSlack : above;
    m += up;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] *= alpha;
    if constexpr (kMod) {
#pragma unroll
      for (int j = 0; j < 2; ++j) sc[j] -= up;
    }
  };
  // K operand i of the scores (i = 2 s + j: k-step s, block j), V operand i of
  // P.V (i = (2 j + ks) * DT + d)
  auto read_k = [&](const uint16_t* tile, int i) VOOM_INLINE {
    return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(tile) +
                                           (i & 1) * (kBlkElems * 2) + (k_lane ^ (32 * (i >> 1))));
  };
  auto read_v = [&](const uint16_t* tile, int i) VOOM_INLINE {
    const int j = i / (2 * DT), ks = (i / DT) & 1, d = i % DT;
    return *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(tile) +
                                           (2 + j) * (kBlkElems * 2) + d * (32 * kBlk * 2) +
                                           v_lane[ks]);
  };

  auto first_scores = [&](const uint16_t* tile, Scores& sc) VOOM_INLINE {
#pragma unroll
    for (int j = 0; j < 2; ++j) sc[j] = f32x16{};
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i) {
      sc[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          __builtin_bit_cast(bf16x8, read_k(tile, i)), __builtin_bit_cast(bf16x8, qop[i >> 1]),
          sc[i & 1], 0, 0, 0);
    }
  };
  // Bits of the V operand's dwords (16-key step jk of tile t) that hold tokens
  // of the sequence.
  auto tail_mask = [&](int t, int jk, uint32_t (&keep)[4]) VOOM_INLINE {
    const int lim = ctx - t * kKeys - 16 * jk - 8 * lh;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      keep[e] = (2 * e < lim ? 0xffffu : 0u) | (2 * e + 1 < lim ? 0xffff0000u : 0u);
  };
  // One of P's pairs, into the operand layout, rounded to bf16 for the matrix units; the
  // normaliser, and with it the LSE, sums the unrounded weights.
  auto form_p = [&](int e, const Scores& sc, u32x4 (&pk)[2][2]) VOOM_INLINE {
    const int j = e >> 3, i = 2 * (e & 7);
    float p0, p1;
    if constexpr (kMod) {
      p0 = fast_exp2(sc[j][i]);
      p1 = fast_exp2(sc[j][i + 1]);
    } else {
      p0 = fast_exp2(__builtin_fmaf(sc[j][i], a.scale, -m));
      p1 = fast_exp2(__builtin_fmaf(sc[j][i + 1], a.scale, -m));
    }
    pk[j][i >> 3][(i & 7) >> 1] = pack_bf16x2(p0, p1);
    l += p0 + p1;
  };

  // Tile t (the key tile of stage c), of which and of the next every row of the wavefront
  // sees all: scores of the next on the matrix cores while the vector units form P, then
  // P.V while they turn those scores into logits and find their maximum.  The next stage's
  // loads go out one by one between the MFMAs.
  auto whole_tile = [&](int t, const uint16_t* tile, uint16_t* next, const Scores& sc,
                        Scores& nx) VOOM_INLINE {
    u32x4 pk[2][2];
    u32x4 ring[kAhead];
#pragma unroll
    for (int j = 0; j < 2; ++j) nx[j] = f32x16{};
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ring[i] = read_k(tile, i);
    __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i) {
      nx[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          __builtin_bit_cast(bf16x8, ring[i % kAhead]), __builtin_bit_cast(bf16x8, qop[i >> 1]),
          nx[i & 1], 0, 0, 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
      if (i + kAhead < 2 * KS) {
        ring[i % kAhead] = read_k(tile, i + kAhead);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
      }
      if (i * kLoads / (2 * KS) != (i + 1) * kLoads / (2 * KS)) {
        load_piece(i * kLoads / (2 * KS), next);
        __builtin_amdgcn_sched_group_barrier(kVmemRead, 1, 0);
      }
#pragma unroll
      for (int e = i * 16 / (2 * KS); e < (i + 1) * 16 / (2 * KS); ++e) {
        form_p(e, sc, pk);
        __builtin_amdgcn_sched_group_barrier(kValu, kMod ? 0 : 2, 0);
        __builtin_amdgcn_sched_group_barrier(kTrans, 2, 0);
        __builtin_amdgcn_sched_group_barrier(kValu, 3, 0);
      }
    }
    // (the weights are formed here: not behind the branch of cap_far)
#pragma unroll
    for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(pk[e >> 1][e & 1]), "+v"(l));
    __builtin_amdgcn_sched_barrier(0);
    const float add0 =
        (BIAS ? slope * static_cast<float>((t + 1) * kKeys + 8 * lh - sight.at) : 0.f) - m;
    auto add_of = [&](int j, int i) VOOM_INLINE {
      if constexpr (!BIAS) return add0;
      return __builtin_fmaf(slope, static_cast<float>(key_of(j, i)), add0);
    };
    const Poly poly = cap_far(nx);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ring[i] = read_v(tile, i);
    __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 1);
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * DT; ++i) {
      const int j = i / (2 * DT), ks = (i / DT) & 1, d = i % DT;
      acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ring[i % kAhead]),
                                                       __builtin_bit_cast(bf16x8, pk[j][ks]),
                                                       acc[d], 0, 0, 0);
      __builtin_amdgcn_sched_group_barrier(kMfma, 1, 1);
      if (i + kAhead < 4 * DT) {
        ring[i % kAhead] = read_v(tile, i + kAhead);
        __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 1);
      }
#pragma unroll
      for (int e = i * 16 / (4 * DT); e < (i + 1) * 16 / (4 * DT); ++e) {
        if constexpr (kMod) {
          nx[0][e] = logit(nx[0][e], poly, add_of(0, e));
          nx[1][e] = logit(nx[1][e], poly, add_of(1, e));
          __builtin_amdgcn_sched_group_barrier(kValu, 2 * ((CAP ? 5 : 1) + (BIAS ? 1 : 0)), 1);
        }
        mx = fmaxf(fmaxf(mx, nx[0][e]), nx[1][e]);
        __builtin_amdgcn_sched_group_barrier(kValu, 1, 1);
      }
    }
    raise(mx, nx);
  };

  // Any tile t (stage c) that some row of the wavefront sees: its scores are in sc, which
  // then takes those of the next one if a row sees that too.
  auto edge_tile = [&](int c, const uint16_t* tile, Scores& sc, auto careful) VOOM_INLINE {
    const int t = keys.tile(c);
    u32x4 pk[2][2];
#pragma unroll
    for (int e = 0; e < 16; ++e) form_p(e, sc, pk);
    // Tokens past the sequence's end are garbage and are cut out of V^T.  Keys that a row does
    // not see have P = 0 in that row, but 0 times a NaN or an infinity is NaN: then `careful`.
    auto values = [&](auto masked) VOOM_INLINE {
#pragma unroll
      for (int jk = 0; jk < 4; ++jk) {
        uint32_t keep[4];
        if constexpr (masked.value) tail_mask(t, jk, keep);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          u32x4 vv = read_v(tile, jk * DT + d);
          if constexpr (masked.value) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vv[e] &= keep[e];
          }
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, vv), __builtin_bit_cast(bf16x8, pk[jk >> 1][jk & 1]),
              acc[d], 0, 0, 0);
        }
        if constexpr (masked.value) __builtin_amdgcn_sched_barrier(0);
      }
    };
    if constexpr (!careful.value) {
      if ((t + 1) * kKeys > ctx) values(std::true_type{});
      else values(std::false_type{});
    } else {
      // Key by key: V^T with one key's column alone times P^T, added only to
      // the rows that see the key.
#pragma unroll
      for (int jk = 0; jk < 4; ++jk) {
#pragma unroll 1
        for (int k = 0; k < 16; ++k) {
          const int kt = t * kKeys + 16 * jk + k;
          if (kt >= ctx) break;
          const bool sees = (kt >= lo && kt < hi) || kt < prefix;
          const int at = lh == (k >> 3) ? (k & 7) : -1;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            u32x4 vv = read_v(tile, jk * DT + d);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              vv[e] &= (at == 2 * e ? 0xffffu : 0u) | (at == 2 * e + 1 ? 0xffff0000u : 0u);
            const f32x16 one = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                __builtin_bit_cast(bf16x8, vv), __builtin_bit_cast(bf16x8, pk[jk >> 1][jk & 1]),
                f32x16{}, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] += sees ? one[e] : 0.f;
            __builtin_amdgcn_sched_barrier(0);  // one product in registers at a time
          }
        }
      }
    }
  };
  // Scores of stage c's key tile, if a row of the wavefront sees it.
  auto edge_scores = [&](int c, const uint16_t* tile, Scores& sc) VOOM_INLINE {
    const int t = keys.tile(c);
    if (!any_sees(t)) return;
    first_scores(tile, sc);
    mask_scores(t, sc);
    raise(max_of(sc), sc);
  };

  Scores sc_a, sc_b;
  // Stage c has landed for every wavefront and the other buffer is no longer read.
  auto landed = [&]() VOOM_INLINE {
    wait_vmem_all();
    lds_barrier();
  };
  // The stages of tiles that every row of the wavefront sees whole, [whole, whole_end): the
  // first at an even distance from the piece's start (an edge tile may be a whole one).  All
  // wavefronts pass one barrier a stage, whichever loop they are in.
  int whole = (lo_max + kKeys - 1) / kKeys - keys.gap;
  whole = whole > c_lo ? whole + ((whole - c_lo) & 1) : c_lo;
  const int whole_end = has_rows ? hi_min / kKeys - keys.gap : 0;
  int c;
  auto edges = [&](int end, auto careful) VOOM_INLINE {
    for (; c < end; c += 2) {
      landed();
      if (c + 1 < c_hi) load_stage(c + 1, tile_b);
      if (any_sees(keys.tile(c))) edge_tile(c, tile_a, sc_a, careful);
      if (c + 1 >= c_hi) {
        c = c_hi;
        return;
      }
      edge_scores(c + 1, tile_a, sc_a);
      landed();
      if (c + 2 < c_hi) load_stage(c + 2, tile_a);
      if (any_sees(keys.tile(c + 1))) edge_tile(c + 1, tile_b, sc_a, careful);
      if (c + 2 < c_hi) edge_scores(c + 2, tile_b, sc_a);
    }
  };
  auto start = [&]() VOOM_INLINE {
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x16{};
    m = 0.f;
    above = -FLT_MAX;
    l = 0.f;
    c = c_lo;
    win = -kWave;
    // (what the first tile needs is formed for it, not kept in registers for a second walk)
    asm volatile("" : "+s"(c));
    if (c < c_hi) {
      // K of the first tile, then (in flight while it is scored) the first stage
      stage_blocks(c - 1);
#pragma unroll
      for (int i = 0; i < kLoads / 2; ++i) load_piece(i, tile_b);
      load_q();
      load_stage(c, tile_a);
      static_assert(kLoads == 8 || kLoads == 4, "the wait below counts the first stage's loads");
      // gfx9 encoding: vmcnt kLoads, expcnt 7, lgkmcnt 15
      if constexpr (kLoads == 8) __builtin_amdgcn_s_waitcnt(0x0F78);
      else __builtin_amdgcn_s_waitcnt(0x0F74);
      lds_barrier();
      edge_scores(c, tile_b, sc_a);
    }
  };
  // A piece is walked as if no value that a row does not see were NaN or infinite.  Where its
  // sums end so, it is walked once more, every tile key by key.
  if (threadIdx.x == 0) again = 0;
  start();
#pragma unroll 1
  for (int phase = 0; phase < 2; ++phase) {
    edges(phase == 0 && whole + 2 < whole_end && whole + 2 < c_hi ? whole : c_hi,
          std::false_type{});
    // (pairs, the tile after them included: its scores run ahead)
    for (; c + 2 < c_hi && c + 3 <= whole_end && c >= whole; c += 2) {
      landed();
      stage_blocks(c + 1);
      whole_tile(keys.tile(c), tile_a, tile_b, sc_a, sc_b);
      landed();
      stage_blocks(c + 2);
      whole_tile(keys.tile(c + 1), tile_b, tile_a, sc_b, sc_a);
    }
  }
  if (c_lo < c_hi) {
    float odd = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int i = 0; i < 16; ++i) odd = __builtin_fmaf(acc[d][i], 0.f, odd);
    }
    if (__builtin_amdgcn_ballot_w64(odd != 0.f) != 0) again = 1;
    lds_barrier();  // (the buffers are no longer read either)
    if (uniform(again) != 0) {
      start();
      edges(c_hi, std::true_type{});
    }
  }

  const float lt = l + __shfl_xor(l, 32);
  // (a padded sequence's rows behind its new tokens are written here too)
  const int t_row = row / a.G;
  const int row_head = kvh * a.G + (row - t_row * a.G);
  if (slot < 0) {
    if (a.starts != nullptr ? row >= R : t_row >= a.T) return;
    const bool empty = row >= R || lt == 0.f;
    const float inv = 1.f / lt;
    const size_t at = out_at(a, b, base, t_row, row_head);
    uint16_t* o = a.out + at * D + 4 * lh;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *reinterpret_cast<u32x2*>(o + 32 * d + 8 * i) =
            empty ? u32x2{0u, 0u}
                  : u32x2{pack_bf16x2(acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv),
                          pack_bf16x2(acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv)};
      }
    }
    if (lh == 0 && a.lse != nullptr)
      a.lse[at] = empty ? -INFINITY : (m + __log2f(lt)) * 0.6931471805599453f;
    return;
  }
  if (row >= R) return;  // (not merged)
  const size_t p = (static_cast<size_t>(kvh) * wa.p.slots + slot) * kTileRows + w * kRows + l32;
  float* o = a.part_o + p * D + 4 * lh;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<f32x4*>(o + 32 * d + 8 * i) =
          f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
    }
  }
  if (lh == 0) *reinterpret_cast<float2*>(a.part_ml + p * 2) = {lt == 0.f ? -FLT_MAX : m, lt};
}

// Merges the pieces of cut row tiles, a row to D / 4 lanes, a few rows of one to a workgroup, so
// that all loads of a row are on their way at once (504 row tiles in two pieces each: 17 us, a
// wavefront a row at a time 33).
constexpr int kJoinThreads = 256;
constexpr int kJoinGroups = 2048;

template <int D>
__global__ __launch_bounds__(kJoinThreads) void gqa_chunk_join_kernel(WideArgs wa) {
  constexpr int kLanes = D / 4;
  constexpr int kAtOnce = kJoinThreads / kLanes;  // rows
  constexpr int kTogether = 8;                    // pieces in flight
  constexpr int kEach = kTileRows / kAtOnce;      // workgroups' shares of a row tile
  const ChunkArgs& a = wa.c;
  const int dim = static_cast<int>(threadIdx.x) % kLanes * 4;
  const int all = wa.head[0] * a.NKV * kEach;
  for (int at = static_cast<int>(blockIdx.x); at < all; at += kJoinGroups) {
    const int pair = at / kEach;
    const int k = pair / a.NKV, kvh = pair - k * a.NKV;
    const int4 cut = wa.cuts[2 * k], seq = wa.cuts[2 * k + 1];
    const int b = uniform(cut.x), rt = uniform(cut.y), parts = uniform(cut.z);
    const int n = uniform(seq.x), base = uniform(seq.y);
    const int r = (at - pair * kEach) * kAtOnce + static_cast<int>(threadIdx.x) / kLanes;
    const int row = rt * kTileRows + r;
    const int tok = row / a.G;
    if (tok >= n && (a.starts != nullptr || tok >= a.T)) continue;
    const size_t first =
        (static_cast<size_t>(kvh) * wa.p.slots + uniform(cut.w)) * kTileRows + r;
    float M = -FLT_MAX, L = 0.f;
    f32x4 acc = {};
    for (int s0 = 0; s0 < parts && tok < n; s0 += kTogether) {
      float2 ml[kTogether];
      f32x4 v[kTogether];
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        if (u > 0 && s0 + u >= parts) break;
        const size_t p = first + static_cast<size_t>(s0 + u) * kTileRows;
        ml[u] = *reinterpret_cast<const float2*>(a.part_ml + p * 2);
        v[u] = *reinterpret_cast<const f32x4*>(a.part_o + p * D + dim);
      }
      float mn = M;
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        if (u > 0 && s0 + u >= parts) break;
        mn = fmaxf(mn, ml[u].x);
      }
      const float f = fast_exp2(M - mn);
      M = mn;
      L *= f;
      acc *= f;
#pragma unroll
      for (int u = 0; u < kTogether; ++u) {
        if (u > 0 && s0 + u >= parts) break;
        const float ws = fast_exp2(ml[u].x - mn);
        L += ml[u].y * ws;
        acc += v[u] * ws;
      }
    }
    const bool empty = tok >= n || L == 0.f;
    const float inv = 1.f / L;
    const size_t out_row = out_at(a, b, base, tok, kvh * a.G + (row - tok * a.G));
    *reinterpret_cast<u32x2*>(a.out + out_row * D + dim) =
        empty ? u32x2{0u, 0u}
              : u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv),
                      pack_bf16x2(acc[2] * inv, acc[3] * inv)};
    if (dim == 0 && a.lse != nullptr)
      a.lse[out_row] = empty ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
  }
}

size_t up(size_t bytes) { return (bytes + 255) & ~size_t(255); }

template <int D, bool CAP>
void launch_tiles(const WideArgs& w, bool bias, dim3 grid, hipStream_t stream) {
  if (bias)
    hipLaunchKernelGGL((gqa_chunk_tiles_kernel<D, CAP, true>), grid, dim3(NW * kWave), 0, stream,
                       w);
  else
    hipLaunchKernelGGL((gqa_chunk_tiles_kernel<D, CAP, false>), grid, dim3(NW * kWave), 0, stream,
                       w);
}

}  // namespace

// A piece of a cut row tile has more than half of the shortest candidate's key tiles, of which
// all workers' shares hold workers / kCaps[last]: at most twice as many pieces, all heads
// together, and half as many cut row tiles.
WidePlan plan_wide(int B, int NKV, int D, int G, int N, int T, long long tokens) {
  WidePlan p;
  p.workers = 2 * device_cu_count();
  const long long entries =
      N > 0 ? static_cast<long long>(N) * G / kTileRows + (B < N ? B : N)
            : B * ((static_cast<long long>(T) * G + kTileRows - 1) / kTileRows);
  p.entries = static_cast<int>(entries);
  p.cuts = static_cast<int>(p.workers / kCaps[kTries - 1] / NKV) + 1;
  // (nor more than pieces of kMinPiece key tiles or a little under)
  const long long parts = (tokens / kKeys + 1) / (kMinPiece / 2) + 1;
  if (p.cuts > entries) p.cuts = p.entries;
  p.slots = static_cast<int>(2LL * (p.workers / kCaps[kTries - 1] / NKV + 1));
  if (p.slots > parts * entries) p.slots = static_cast<int>(parts * entries);
  p.pieces = p.entries + p.slots;
  const size_t rows = static_cast<size_t>(p.slots) * NKV * kTileRows;
  p.bytes = up(rows * D * sizeof(float)) + up(rows * sizeof(float2)) +
            up(2 * p.pieces * sizeof(int4)) + up(2 * p.cuts * sizeof(int4)) + 256 +
            up(p.entries * sizeof(int32_t));
  return p;
}

int launch_wide(const ChunkArgs& a, const WidePlan& p, int D, void* workspace,
                hipStream_t stream) {
  WideArgs w;
  w.c = a;
  w.p = p;
  const size_t rows = static_cast<size_t>(p.slots) * a.NKV * kTileRows;
  char* at = static_cast<char*>(workspace);
  w.c.part_o = reinterpret_cast<float*>(at);
  at += up(rows * D * sizeof(float));
  w.c.part_ml = reinterpret_cast<float*>(at);
  at += up(rows * sizeof(float2));
  w.pieces = reinterpret_cast<int4*>(at);
  at += up(2 * p.pieces * sizeof(int4));
  w.cuts = reinterpret_cast<int4*>(at);
  at += up(2 * p.cuts * sizeof(int4));
  w.head = reinterpret_cast<int32_t*>(at);
  at += 256;
  w.lengths = reinterpret_cast<int32_t*>(at);
  hipLaunchKernelGGL(gqa_chunk_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, w);
  int rc = VOOM_LAUNCH_CHECK("paged_gqa_chunk: plan launch");
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>(static_cast<long long>(p.pieces) * a.NKV));
  const bool bias = a.slopes != nullptr || (a.cap == 0.f && !(a.scale > 0.f));
  if (D == 128) {
    if (a.cap != 0.f) launch_tiles<128, true>(w, bias, grid, stream);
    else launch_tiles<128, false>(w, bias, grid, stream);
  } else {
    if (a.cap != 0.f) launch_tiles<64, true>(w, bias, grid, stream);
    else launch_tiles<64, false>(w, bias, grid, stream);
  }
  rc = VOOM_LAUNCH_CHECK("paged_gqa_chunk: tiles launch");
  if (rc) return rc;
  const dim3 jgrid(kJoinGroups);
  if (D == 128)
    hipLaunchKernelGGL(gqa_chunk_join_kernel<128>, jgrid, dim3(kJoinThreads), 0, stream, w);
  else
    hipLaunchKernelGGL(gqa_chunk_join_kernel<64>, jgrid, dim3(kJoinThreads), 0, stream, w);
  return VOOM_LAUNCH_CHECK("paged_gqa_chunk: join launch");
}

}  // namespace voom
