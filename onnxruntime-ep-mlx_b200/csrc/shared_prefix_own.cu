// shared_prefix_own_kernel: single new tokens and short chunks (at most own_rows = 8 NT rows of a kv
// head) against their sequence's own keys.
//
// Bound by HBM: every own key is read once per call and serves the few rows of its kv head (2 g
// flops per byte).  All own keys of these sequences form one stream of 16-key tiles (sequence, kv
// head, tile); each warp of the persistent grid owns an equal contiguous range of it, so ragged
// lengths balance exactly.  A warp streams its tiles through a private ring of shared-memory stages
// that its lanes fill with asynchronous 16-byte copies (128-byte swizzle), the lookahead running across
// sequence boundaries.  Per tile:
//   S^T[16 keys x 8 NT rows] = K . Q^T       mma.m16n8k16, K by ldmatrix, Q in registers
//   softmax with a running maximum           fp32, exp2 domain
//   O^T[d x 8 NT rows] += V^T . P^T          ldmatrix.trans; P as a hi + lo pair of 16-bit values
// (a 128-row tcgen05 tile would be empty but for these rows and the tensor pipe is not the bound).
// Measured alone, bf16, d 128: 315 MB in 57 us, 1.14 GB in 184 us (6.2 TB/s, 0.95 of a plain copy's rate).
// Beside the tensor-core pass both run slower, but sooner than one after the other.  Not better: stages
// filled by TMA (59 and 188 us), separate stages for K and V (64 us), tiles prefetched to L2 (78 us).
// A (sequence, kv head) segment inside one warp's range goes to the own slab; a cut one leaves a
// triple per warp, at most two per warp, for the merge kernel.
#include <atomic>

#include "b200_tcgen05.cuh"
#include "shared_prefix.cuh"

namespace b200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// 16 bytes global -> shared memory, or 16 zero bytes.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int D>
struct OwnLayout {
  static constexpr int kBoxes = D / 64;
  static constexpr int kBoxBytes = kOwnTile * 128;
  static constexpr int kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kStageBytes = 2 * kTileBytes;  // K and V
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kSmem = kOwnWarps * kStages * kStageBytes;
};

// 16-byte piece `chunk` of tile row `row` in the 128B-swizzled boxes.
__device__ __forceinline__ uint32_t own_swizzle(int row, int chunk) {
  return (uint32_t)((chunk >> 3) * (kOwnTile * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// A part of one (sequence, kv head) segment of the tile stream.
struct Piece {
  int valid, b, kh, t0, t1, tiles, c0, nq, past, total;
  int64_t seg_start;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kOwnWarps, NT == 1 ? 4 : 3) shared_prefix_own_kernel(const __grid_constant__ SharedPrefixArgs a) {
  using L = OwnLayout<D>;
  using MMA = mma_op<T>;
  constexpr int KSTEPS = D / 16, STAGES = L::kStages, RING = STAGES + 1, ROWS = 8 * NT;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Piece ring[kOwnWarps][RING];

  release_dependents();
  const B200SharedPrefixParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t wbase_u32 = smem_u32(smem + warp * STAGES * L::kStageBytes);
  Piece* myring = ring[warp];

  const int KV = p.kv_num_heads, g = a.group, H = p.num_heads;
  // The plan is complete: this grid starts after every CTA of the tensor-core kernel has waited for it.
  const OwnRanges ranges((int64_t)__ldcg(a.seq_tiles + p.batch) * KV, a.own_warps);
  const int64_t gw = (int64_t)blockIdx.x * kOwnWarps + warp;
  const int64_t r0 = gw < ranges.warps ? ranges.start(gw) : 0;
  const int64_t r1 = gw < ranges.warps ? ranges.start(gw + 1) : 0;
  if (r0 >= r1) {
    if (blockIdx.x == gridDim.x - 1) wait_previous();  // as at the end
    return;
  }
  const float qk_scale = p.softcap > 0.f ? p.scale : p.scale * kLog2e;

  // Sequences seq0 .. seq0 + 31, one per lane, so that going on to the next piece needs no loads.
  int seq0 = 0, seq_first = 0, seq_c0 = 0, seq_nq = 0, seq_past = 0, seq_tiles = 0;
  auto load_window = [&](int from) {
    seq0 = from;
    const int b = min(from + lane, p.batch);
    seq_first = __ldcg(a.seq_tiles + b);
    if (b < p.batch) {
      seq_tiles = __ldcg(a.seq_tiles + b + 1) - seq_first;
      seq_c0 = p.cumulative_sequence_length[b];
      seq_nq = p.cumulative_sequence_length[b + 1] - seq_c0;
      seq_past = p.past_seqlens[b];
    }
  };
  // The piece at stream position x (< r1) into ring slot `slot` (the whole warp).
  auto locate = [&](int slot, int64_t x) {
    Piece u{};
    if (x < r1) {
      unsigned before = __ballot_sync(0xffffffffu, (int64_t)seq_first * KV <= x);
      if (before == 0xffffffffu || before == 0) {  // not in the window: 32-way search
        int lo = before ? seq0 : 0, hi = p.batch;  // the largest lo with seq_tiles[lo] * KV <= x
        while (hi - lo > 1) {
          const int step = (hi - lo + 31) / 32, at = lo + lane * step;
          const unsigned le = __ballot_sync(0xffffffffu, at < hi && (int64_t)__ldcg(a.seq_tiles + min(at, p.batch)) * KV <= x);
          lo += (__popc(le) - 1) * step;
          hi = min(hi, lo + step);
        }
        load_window(lo);
        before = __ballot_sync(0xffffffffu, (int64_t)seq_first * KV <= x);
      }
      // sequences without tiles share their successor's offset: the last one not past x owns it
      const int src = 31 - __clz(before);
      const int first = __shfl_sync(0xffffffffu, seq_first, src), tiles = __shfl_sync(0xffffffffu, seq_tiles, src);
      u.b = seq0 + src;
      u.c0 = __shfl_sync(0xffffffffu, seq_c0, src);
      u.nq = __shfl_sync(0xffffffffu, seq_nq, src);
      u.past = __shfl_sync(0xffffffffu, seq_past, src);
      if (tiles > 0) {
        const int64_t rel = x - (int64_t)first * KV;
        u.valid = 1;
        u.kh = (int)OwnRanges::quotient(rel, tiles);
        u.tiles = tiles;
        u.t0 = (int)(rel - (int64_t)u.kh * tiles);
        u.t1 = (int)min((int64_t)tiles, u.t0 + (r1 - x));
        u.seg_start = (int64_t)first * KV + (int64_t)u.kh * tiles;
        u.total = u.past + u.nq;
      }
    }
    __syncwarp();
    if (lane == 0) myring[slot] = u;
    __syncwarp();
  };

  // Producer: tile pt of the piece in ring slot ps goes into stage `issued` % STAGES, 16 bytes per lane
  // and copy; rows without a key (past the sequence's end, or of a block id out of range) become zeros.
  const char* const kv_base[2] = {static_cast<const char*>(p.key_cache), static_cast<const char*>(p.value_cache)};
  const int64_t row_bytes = (int64_t)KV * D * 2;
  int ps = 0, pt = 0, issued = 0, window = 0;
  int32_t window_blk = -1;  // lane i: block of tile window + i of the piece
  bool producing = false, fresh = true;
  auto produce = [&]() {
    while (producing && pt >= myring[ps].t1) {
      const int64_t next = myring[ps].seg_start + myring[ps].t1;
      ps = (ps + 1) % RING;
      locate(ps, next);
      producing = myring[ps].valid != 0;
      pt = myring[ps].t0;
      fresh = true;
    }
    if (producing) {
      const Piece& u = myring[ps];
      if (fresh || pt - window == 32) {
        fresh = false;
        window = pt;
        window_blk = pt + lane < u.t1 ? __ldg(p.block_table + (int64_t)u.b * p.max_blocks_per_seq +
                                              (pt + lane) * kOwnTile / p.block_size)
                                      : -1;
      }
      const int32_t blk = __shfl_sync(0xffffffffu, window_blk, pt - window);
      const int pos = pt * kOwnTile;
      const bool ok = blk >= 0 && blk < p.num_blocks;
      if (!ok && lane == 0) set_status(p.device_status, kStatusBadBlock);
      const int keys = ok ? u.total - pos : 0;
      const int64_t first = ok ? (((int64_t)blk * p.block_size + pos % p.block_size) * KV + u.kh) * D * 2 : 0;
      const uint32_t dst = wbase_u32 + issued % STAGES * L::kStageBytes;
      constexpr int CH = D / 8;  // 16-byte pieces per row
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char* src = kv_base[t] + first + lane / CH * row_bytes + lane % CH * 16;
#pragma unroll
        for (int i = 0; i < kOwnTile * CH / 32; ++i) {
          const int row = i * (32 / CH) + lane / CH;
          cp_async16(dst + t * L::kTileBytes + own_swizzle(row, lane % CH), row < keys ? src : kv_base[t], row < keys);
          src += 32 / CH * row_bytes;
        }
      }
      ++pt;
      ++issued;
    }
    cp_async_commit();  // a group per call, empty at the end
  };
  load_window(0);
  locate(0, r0);
  producing = myring[0].valid != 0;
  pt = myring[0].t0;
  int consumed = 0;
  for (int i = 0; i < STAGES; ++i) produce();

  int cs = 0, ct = myring[0].t0;
  const int col0 = (lane & 3) * 2;  // rows held by this lane: 8 n + col0, + 1

  while (consumed < issued) {
    const Piece u = myring[cs];
    const int rows = u.nq * g;

    // Q^T fragments: column lane / 4 of n-tile n is row 8 n + lane / 4 = (token, head in group)
    uint32_t qf[NT][KSTEPS][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + (lane >> 2), kq = (lane & 3) * 2;
      const bool in = r < rows;
      const T* qrow = static_cast<const T*>(p.query) + (int64_t)(u.c0 + (in ? r / g : 0)) * p.query_row_stride +
                      (int64_t)(u.kh * g + (in ? r % g : 0)) * D;
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        qf[n][kk][0] = in ? *reinterpret_cast<const uint32_t*>(qrow + kk * 16 + kq) : 0u;
        qf[n][kk][1] = in ? *reinterpret_cast<const uint32_t*>(qrow + kk * 16 + 8 + kq) : 0u;
      }
    }
    float m[NT][2], l[NT][2], o[NT][KSTEPS][4];
    int limit[NT][2];  // last own key the row sees; -1: no such row
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + col0 + e;
        m[n][e] = -INFINITY;
        l[n][e] = 0.f;
        limit[n][e] = r < rows ? u.past + r / g : -1;
      }
#pragma unroll
      for (int mt = 0; mt < KSTEPS; ++mt) o[n][mt][0] = o[n][mt][1] = o[n][mt][2] = o[n][mt][3] = 0.f;
    }

    for (; ct < u.t1; ++ct) {
      const int s = consumed % STAGES;
      const int pos0 = ct * kOwnTile;
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      const bool full = pos0 + kOwnTile <= u.past + 1;  // every row sees every key
      const uint32_t kbase = wbase_u32 + s * L::kStageBytes, vbase = kbase + L::kTileBytes;

      float c[NT][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) c[n][j][0] = c[n][j][1] = c[n][j][2] = c[n][j][3] = 0.f;
      {
        const int row = (lane & 7) + ((lane >> 3) & 1) * 8, half = lane >> 4;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; kk += 2) {
          uint32_t af[4], bf[4];
          ldsm_x4(kbase + own_swizzle(row, kk * 2 + half), af[0], af[1], af[2], af[3]);
          ldsm_x4(kbase + own_swizzle(row, kk * 2 + 2 + half), bf[0], bf[1], bf[2], bf[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            MMA::run(c[n][0], af, qf[n][kk][0], qf[n][kk][1]);
            MMA::run(c[n][1], bf, qf[n][kk + 1][0], qf[n][kk + 1][1]);
          }
        }
      }
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float sc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pos = pos0 + (lane >> 2) + ((e >> 1) << 3);
          float x = (c[n][0][e] + c[n][1][e]) * qk_scale;
          if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap) * kLog2e;
          const bool seen = full ? limit[n][e & 1] >= 0 : pos <= limit[n][e & 1];
          sc[e] = seen ? x : -INFINITY;
        }
        float mx0 = fmaxf(sc[0], sc[2]), mx1 = fmaxf(sc[1], sc[3]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
        }
        // The running maximum moves only when a score exceeds it by more than 2^8 (warp-uniform), so P
        // stays within 2^8 and most tiles leave o alone.
        if (__any_sync(0xffffffffu, mx0 > m[n][0] + 8.f || mx1 > m[n][1] + 8.f)) {
          const float mn0 = fmaxf(m[n][0], mx0), mn1 = fmaxf(m[n][1], mx1);
          const float al0 = mn0 == -INFINITY ? 1.f : tc::ex2(m[n][0] - mn0), al1 = mn1 == -INFINITY ? 1.f : tc::ex2(m[n][1] - mn1);
          l[n][0] *= al0;
          l[n][1] *= al1;
          m[n][0] = mn0;
          m[n][1] = mn1;
#pragma unroll
          for (int mt = 0; mt < KSTEPS; ++mt) {
            o[n][mt][0] *= al0; o[n][mt][2] *= al0;
            o[n][mt][1] *= al1; o[n][mt][3] *= al1;
          }
        }
        const float mu0 = m[n][0] == -INFINITY ? 0.f : m[n][0], mu1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
        const float p0 = tc::ex2(sc[0] - mu0), p1 = tc::ex2(sc[1] - mu1);
        const float p2 = tc::ex2(sc[2] - mu0), p3 = tc::ex2(sc[3] - mu1);
        l[n][0] += p0 + p2;
        l[n][1] += p1 + p3;
        // P to 16 bits twice: the rounded value and what the rounding left (about 16 bits in all)
        const uint32_t x0 = MMA::pack(p0, p1), x1 = MMA::pack(p2, p3);
        const float2 h0 = MMA::unpack(x0), h1 = MMA::unpack(x1);
        ph[n][0] = movm_t(x0);
        ph[n][1] = movm_t(x1);
        pl[n][0] = movm_t(MMA::pack(p0 - h0.x, p1 - h0.y));
        pl[n][1] = movm_t(MMA::pack(p2 - h1.x, p3 - h1.y));
      }
      {
        const int jm = lane >> 3;
        const int row = (lane & 7) + (jm >> 1) * 8, sub = jm & 1;
#pragma unroll
        for (int mt = 0; mt < KSTEPS; ++mt) {
          uint32_t af[4];
          ldsm_x4_t(vbase + own_swizzle(row, mt * 2 + sub), af[0], af[1], af[2], af[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            MMA::run(o[n][mt], af, ph[n][0], ph[n][1]);
            MMA::run(o[n][mt], af, pl[n][0], pl[n][1]);
          }
        }
      }
      __syncwarp();
      ++consumed;
      produce();
    }

    // the piece's triples: column sums of l, then the own slab or this warp's rows
    const int dr = lane >> 2;
    const bool whole = u.t0 == 0 && u.t1 == u.tiles;
    // slot 0: the warp's first piece, slot 1: its last one
    const int64_t wrow = (gw * 2 + (u.seg_start + u.t0 == r0 ? 0 : 1)) * ROWS;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l[n][0] += __shfl_xor_sync(0xffffffffu, l[n][0], off);
        l[n][1] += __shfl_xor_sync(0xffffffffu, l[n][1], off);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * n + col0 + e;
        if (r >= rows) continue;
        const int64_t row = whole ? (int64_t)a.splits * a.rows + (int64_t)(u.c0 + r / g) * H + u.kh * g + r % g : wrow + r;
        float* po = (whole ? a.slab_o : a.warp_o) + row * D;
        if (dr == 0) (whole ? a.slab_ml : a.warp_ml)[row] = make_float2(m[n][e], l[n][e]);
#pragma unroll
        for (int mt = 0; mt < KSTEPS; ++mt) {
          po[mt * 16 + dr] = o[n][mt][e];
          po[mt * 16 + dr + 8] = o[n][mt][e + 2];
        }
      }
    }
    cs = (cs + 1) % RING;
    ct = myring[cs].t0;
  }
  // The last CTA stays until the tensor-core kernel is done: the merge, which waits for this grid, then
  // has both.  The others leave their place to this grid's next CTAs.
  if (blockIdx.x == gridDim.x - 1) wait_previous();
}

template <typename T, int D, int NT>
cudaError_t launch_own_t(const SharedPrefixArgs& a, cudaStream_t stream) {
  auto kernel = shared_prefix_own_kernel<T, D, NT>;
  static std::atomic<uint32_t> ready[64];  // per device: attribute set
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!ready[dev & 63].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, OwnLayout<D>::kSmem);
    if (e != cudaSuccess) return e;
    // both kernels' CTAs share an SM only in the largest shared-memory split
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    ready[dev & 63].store(1, std::memory_order_release);
  }
  return launch_dependent(kernel, dim3(a.own_warps / kOwnWarps), dim3(32 * kOwnWarps),
                          OwnLayout<D>::kSmem, stream, a);
}

}  // namespace

cudaError_t launch_shared_prefix_own(const SharedPrefixArgs& a, cudaStream_t stream) {
  const bool bf = a.p.act_dtype == B200_DTYPE_BFLOAT16, wide = a.own_rows > 8;
  if (a.p.head_size == 64) {
    if (bf) return wide ? launch_own_t<__nv_bfloat16, 64, 2>(a, stream) : launch_own_t<__nv_bfloat16, 64, 1>(a, stream);
    return wide ? launch_own_t<__half, 64, 2>(a, stream) : launch_own_t<__half, 64, 1>(a, stream);
  }
  if (bf) return wide ? launch_own_t<__nv_bfloat16, 128, 2>(a, stream) : launch_own_t<__nv_bfloat16, 128, 1>(a, stream);
  return wide ? launch_own_t<__half, 128, 2>(a, stream) : launch_own_t<__half, 128, 1>(a, stream);
}

}  // namespace b200
