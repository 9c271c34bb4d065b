// What the kernels share that stream a paged cache through a ring of stages in LDS
// (gqa_tree.hip, gqa_observe.hip): how units of work are dealt out to workgroups, and
// the loads of a block.
#pragma once

#include "common.h"

namespace voom {

constexpr int kBlk = 32;  // tokens of a K/V block in the pool

typedef __attribute__((address_space(3))) void lds_void;

// Units 0 .. U - 1 over at most W workgroups, as evenly as it goes: the first `rem` of
// them take base + 1, the others base.
struct Split {
  int We, base, rem;
  __device__ __forceinline__ Split(int U, int W) {
    We = U < 1 ? 1 : (U < W ? U : W);
    base = U / We;
    rem = U - base * We;
  }
  __device__ __forceinline__ int begin(int w) const { return w * base + (w < rem ? w : rem); }
  // the workgroup that holds unit u
  __device__ __forceinline__ int group(int u) const {
    const int u_rem = rem * (base + 1);
    return u < u_rem ? u / (base + 1) : rem + (u - u_rem) / base;
  }
};

// The pages of one (sequence, kv head) that a wavefront walks, 64 slots at a time in its
// lanes.
struct Pages {
  const int32_t* row;  // the sequence's table row
  int max_pages, num_slots, nkv, kvh;
  int sub_shift;       // log2 of a page's blocks
  int last;            // the context's last block
  int base, tab;       // first page of those in the lanes, and their slots

  __device__ __forceinline__ Pages(const int32_t* row_, int max_pages_, int num_slots_, int nkv_,
                                   int kvh_, int sub_shift_, int last_)
      : row(row_), max_pages(max_pages_), num_slots(num_slots_), nkv(nkv_), kvh(kvh_),
        sub_shift(sub_shift_), last(last_), base(-(1 << 30)), tab(0) {}

  // Makes sure that the lanes hold the pages of blocks bi .. bi + n - 1 (of those past
  // the last one: its page).
  __device__ __forceinline__ void hold(int bi, int n, int lane) {
    const int first = bi < last ? bi : last;
    if (first >> sub_shift < base || (first + n - 1) >> sub_shift >= base + kWave) {
      base = first >> sub_shift;
      const int p = base + lane;
      tab = p < max_pages ? row[p] : 0;
      wait_vmem_all();  // here, not at the readlanes of every block
    }
  }
  // Pool block (in units of 32 tokens of one kv head) of block bi, the last one for those
  // past it; slot ids outside the pool read slot 0.
  __device__ __forceinline__ size_t block(int bi) const {
    const int at = bi < last ? bi : last;
    const int page = at >> sub_shift;
    int slot = __builtin_amdgcn_readlane(tab, page - base);
    if (static_cast<unsigned>(slot) >= static_cast<unsigned>(num_slots)) slot = 0;
    return ((static_cast<size_t>(slot) * nkv + kvh) << sub_shift) + (at - (page << sub_shift));
  }
};

// One load of 1 KiB, straight into LDS (64 lanes, 16 bytes each, consecutive there): the
// lanes' bytes at `src` of a block of `bytes` bytes; past them zeros.
template <int AUX>
__device__ __forceinline__ void load_piece(const uint16_t* block, int bytes, int src,
                                           uint16_t* to) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(block), static_cast<short>(0), bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)to, 16, src, 0, 0, AUX);
}

}  // namespace voom
