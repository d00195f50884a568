// Shared pieces of the fast path of b200_shared_prefix_attention: its plan in the workspace, the
// argument block and programmatic dependent launch.
//
// One call is four launches:
//   shared_prefix_plan_kernel   lengths -> work lists (1 CTA) and, for bf16 calls of many tokens, an fp16 copy of
//                               the prefix's values (2 CTAs per SM), while the tensor-core pass starts
//   shared_prefix_tc_kernel     tensor-core pass (tcgen05): every token against a range of the
//                               prefix's keys, and long chunks against their own keys
//   shared_prefix_own_kernel    single tokens and short chunks against their own keys (memory bound)
//   shared_prefix_merge_kernel  joins the softmax triples (m, l, o) of each (token, head) row
// The passes leave unnormalised fp32 o with m (log2 domain) and l: prefix range s of the S ranges in
// slab s, own keys in slab S, each slab [num_tokens * num_heads][head_size]; own keys that stream-K
// cut between warps stay in the warps' own rows until the merge.
#pragma once

#include <utility>

#include "b200_common.cuh"
#include "layer_kernels.h"

namespace b200 {

struct SharedPrefixArgs {
  B200SharedPrefixParams p;
  int group;         // query heads per kv head
  int tile_tokens;   // tokens of one 128-row query tile: 128 / group
  int splits;        // S: key ranges of the prefix
  int split_tiles;   // 128-key tiles per range
  int query_pairs;   // pairs of query tiles over all tokens
  int own_rows;      // sequences of at most this many (token, head-in-group) rows: own kernel
  int own_warps;     // warps of the own kernel's grid
  int64_t rows;      // num_tokens * num_heads
  int beside;        // tensor-core CTAs leave room for the own kernel's
  // fp16 copy of the prefix's values (bf16 calls whose copy pays: see shared_prefix_plan_kernel)
  __half* v_copy;    // [prefix_length][kv heads][head_size], or null
  uint64_t* v_inexact;  // [copy_ctas] kv heads (bit: head % 64) of which the CTA met a value that fp16 does not hold
  int copy_ctas;
  // plan
  int* seq_tiles;    // [batch + 1] exclusive prefix of 16-key tiles (per kv head), own kernel
  int* seq_pairs;    // [batch + 1] exclusive prefix of query-tile pairs, tensor-core kernel
  int4* token_info;  // [num_tokens] of a token's sequence: first token, tokens (-1: none valid), first
                     // 16-key tile of the own kernel, tiles (0: own keys on the tensor-core kernel)
  uint32_t* next_item;  // tensor-core items handed out beyond each CTA's first
  // partials
  float* slab_o;     // [splits + 1][rows][head_size]
  float2* slab_ml;   // [splits + 1][rows]
  float* warp_o;     // [own_warps * 2][own_rows][head_size]
  float2* warp_ml;   // [own_warps * 2][own_rows]
};

struct SharedPrefixMaps {
  CUtensorMap k_map, v_map;  // [num_blocks * block_size, kv heads, d]: box {64, 1, 16}
  CUtensorMap q_map;         // [tokens, heads, d]: box {64, group, tile_tokens}
  CUtensorMap vc_map;        // v_copy: box {64, 1, 128}
};

constexpr int kOwnTile = 16;  // keys per tile of the own kernel
constexpr int kOwnWarps = 4;  // warps per CTA
constexpr int kOwnCtasPerSm = 3;  // its shared memory, 65 KB per CTA, leaves room for three
constexpr int kPrefixKeys = 128;  // keys per tile of the tensor-core kernel
constexpr float kCopyScaleLog2 = 11.f, kCopyScale = 2048.f;  // factor on the values of v_copy, taken out of the pass's triples

cudaError_t launch_shared_prefix_tc(const SharedPrefixArgs& a, const SharedPrefixMaps& maps, int num_sms,
                                    cudaStream_t stream);
cudaError_t launch_shared_prefix_own(const SharedPrefixArgs& a, cudaStream_t stream);

// Stream-K ranges of the own kernel: T tiles over W warps, the first `extra` warps own `each` + 1
// consecutive tiles and the others `each`.
struct OwnRanges {
  int64_t total, extra;
  int64_t each;
  int64_t warps;
  __device__ __forceinline__ OwnRanges(int64_t tiles, int grid_warps) : total(tiles) {
    const int64_t most = (tiles + 1) / 2;  // at least 2 tiles per warp: more pieces cost the merge more
    warps = most < 1 ? 1 : (most < grid_warps ? most : grid_warps);
    each = quotient(tiles, warps);
    extra = tiles - each * warps;
  }
  __device__ __forceinline__ int64_t start(int64_t w) const { return w * each + (w < extra ? w : extra); }
  __device__ __forceinline__ int64_t warp_of(int64_t tile) const {
    const int64_t split = extra * (each + 1);
    return tile < split ? quotient(tile, each + 1) : extra + quotient(tile - split, each);
  }
  // 32-bit where it fits: a 64-bit division takes several times as long
  static __device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
    return x < (int64_t)1 << 31 ? (int64_t)((uint32_t)x / (uint32_t)y) : x / y;
  }
};

// Programmatic dependent launch: a kernel launched with the attribute may start once every CTA of
// the previous one has called release_dependents() (or exited); wait_previous() returns when the
// previous kernel has completed and its writes are visible.
__device__ __forceinline__ void release_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
}

}  // namespace b200
