// Matrix products grouped by adapter copy with ragged rows (tcgen05, bf16 operands, fp32 sums).
//
//   MODE 0   y_i  = alpha x_i W_g(i) (+ y_i)       rows i of group g are [o_g, o_{g+1})
//   MODE 1   dW_g = alpha X_g^T dY_g (+ dW_g)      the gradient in the weights
//
// The row offsets live on the device: every CTA scans them once (clamped to the rows there
// are and made monotone, so that no offset can lead out of bounds or to two owners of a row)
// and finds its tiles by binary search. A group may be empty; its dW is zero. In MODE 0 rows
// outside every group are left as they were, or zeroed where the caller asks.
//
// A tile is 128 x BN: MODE 0 128 rows of one group, MODE 1 128 features of the wider operand.
// Ten warps:
//   warp 0     TMA producer (one lane): 64-wide k-steps of A and B into a ring of stages
//   warp 1     TMEM owner and MMA issuer (kind::f16, M = 128, N = BN), two accumulators
//   warps 2-9  epilogue: TMEM -> registers -> (staged, coalesced) stores
// A tile that reaches past its group reads the neighbour's rows: harmless in MODE 0 (each
// output row depends on its own input row; rows past the group are not stored), and cleared
// in shared memory before the last k-step's MMAs in MODE 1, where they would be summed.
//
// fp32 outputs: the tensor core's accumulator rounds towards zero, which shows after some
// hundred additions; every kChunk k-steps the epilogue therefore takes the accumulator into
// registers and adds the chunks with rounding to nearest. bf16 outputs (half a step 2^-9 of
// the value) do not need it.
//
// Few tiles (narrow outputs): a cluster of 2, 4 or 8 CTAs splits the contraction; each CTA
// sends its partial tile to the CTA that owns the rows through distributed shared memory, and
// the owner adds the partials in rank order. No atomics: results are the same on every run.
//
// Every mbarrier wait gives up after ~1 s, sets the error word, and lets each role finish its
// own copies before the CTA frees its TMEM.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "dsmz_ptx.cuh"
#include "dsmz_tcgen05.cuh"

namespace dsmz {
namespace gr {

using tc::kBK;
using tc::kBM;

constexpr int kMaxGroups = 1024;
constexpr int kEpiWarps = 8;
constexpr int kThreadsG = 64 + 32 * kEpiWarps;
constexpr int kChunk = 8;               // k-steps (512 products) an accumulator takes for fp32 outputs
constexpr int kStagePitch = 80;         // bytes of a staged 64-byte row piece (conflict-free 16-byte accesses)
constexpr int kABytes = kBM * kBK * 2;

struct Args {
  const int32_t* offsets;               // G + 1, device
  int32_t G, mode;
  int64_t M;                            // rows of x
  int32_t mdim, ndim, kdim;             // MODE 0: -, N, K; MODE 1: wide, narrow, -
  int32_t bn;                           // MMA N (multiple of 16) = columns of a tile
  int32_t ntn, mtn;                     // column tiles; MODE 1: feature tiles
  int32_t b_mn;                         // MODE 0: W is contiguous along N
  int32_t arows;                        // MODE 0: rows of an A box
  int32_t stages, split;
  int32_t chunk;                        // k-steps per accumulator
  void* out;
  int64_t ld, gstride;                  // output pitch; MODE 1: elements between groups
  int32_t transposed;                   // MODE 1: element (m, n) at n * ld + m
  int32_t out_f32, accumulate, zero_rest, vec;
  float alpha;
};

// 32 lanes x 32 consecutive fp32 columns of TMEM.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Box {inner, rows, 1} of a 3-D tensor map (inner, row, group) into this CTA's shared memory.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_remote(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Bounded wait with cluster-scope acquire (arrivals come from other CTAs).
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, int* err) {
  const uint64_t t0 = gtimer();
  uint64_t tchk = t0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, "
        "p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(kSuspendNs)
        : "memory");
    if (ok) return true;
    const uint64_t t = gtimer();
    if (t - tchk > kPollNs) {
      tchk = t;
      if (*reinterpret_cast<volatile int*>(err) != 0) return false;
      if (t - t0 > kTimeoutNs) {
        atomicExch(err, 1);
        return false;
      }
    }
  }
}

// Row boundaries bnd[0..G+2] = 0, the offsets (clamped to [0, M], running maximum), M; segment
// s = rows [bnd[s], bnd[s+1]): 1..G are the groups, 0 and G+1 the rows outside them. tile0[s] =
// 128-row tiles before segment s (0 and G+1 have none unless they are zeroed). One warp.
__device__ __forceinline__ void scan_groups(const int32_t* off, int G, int M, bool rest, int32_t* bnd, int32_t* tile0,
                                            int lane) {
  int carry = 0;
  for (int i0 = 0; i0 <= G; i0 += 32) {
    const int i = i0 + lane;
    int v = i <= G ? min(max(off[i], 0), M) : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v = max(v, u);
    }
    v = max(v, carry);
    if (i <= G) bnd[i + 1] = v;
    carry = __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) { bnd[0] = 0; bnd[G + 2] = M; }
  __syncwarp();
  int base = 0;
  for (int s0 = 0; s0 < G + 2; s0 += 32) {
    const int s = s0 + lane;
    int n = 0;
    if (s < G + 2 && (rest || (s >= 1 && s <= G))) n = (bnd[s + 1] - bnd[s] + kBM - 1) / kBM;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (s < G + 2) tile0[s] = base + inc - n;
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) tile0[G + 2] = base;
}

struct Tile {
  int seg;                              // segment (MODE 0) or group (MODE 1)
  int m0, n0;                           // first row / feature and first column
  int valid;                            // rows / features of the tile that exist
  int r0, cnt;                          // MODE 1: the group's rows
  int nk;                               // k-steps of the whole contraction
};

template <int MODE>
__device__ __forceinline__ Tile tile_of(const Args& a, const int32_t* bnd, const int32_t* tile0, int t) {
  Tile x;
  if (MODE == 0) {
    int lo = 0, hi = a.G + 1;           // the last segment whose first tile is at or before t
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tile0[mid] * a.ntn <= t) lo = mid; else hi = mid - 1;
    }
    const int nm = tile0[lo + 1] - tile0[lo];
    const int local = t - tile0[lo] * a.ntn;
    const int nt = local / nm, mt = local - nt * nm;   // rows first: concurrent tiles share W's columns
    x.seg = lo;
    x.m0 = bnd[lo] + mt * kBM;
    x.n0 = nt * a.bn;
    x.valid = min(kBM, bnd[lo + 1] - x.m0);
    x.r0 = x.cnt = 0;
    x.nk = (lo >= 1 && lo <= a.G) ? (a.kdim + kBK - 1) / kBK : 0;
  } else {
    const int per = a.mtn * a.ntn;
    x.seg = t / per;
    const int local = t - x.seg * per;
    const int nt = local / a.mtn;
    x.m0 = (local - nt * a.mtn) * kBM;
    x.n0 = nt * a.bn;
    x.valid = min(kBM, a.mdim - x.m0);
    x.r0 = bnd[x.seg + 1];
    x.cnt = bnd[x.seg + 2] - x.r0;
    x.nk = (x.cnt + kBK - 1) / kBK;
  }
  return x;
}

// Four consecutive output columns: (old +) alpha v, rounded once.
__device__ __forceinline__ void put4(const Args& a, char* row, int col, int ncols, float4 v) {
  if (a.out_f32) {
    float* p = reinterpret_cast<float*>(row) + col;
    if (a.vec && ncols >= 4) {
      if (a.accumulate) {
        const float4 o = *reinterpret_cast<const float4*>(p);
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
      }
      *reinterpret_cast<float4*>(p) = v;
    } else {
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) if (c < ncols) p[c] = a.accumulate ? p[c] + x[c] : x[c];
    }
  } else {
    __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(row) + col;
    float x[4] = {v.x, v.y, v.z, v.w};
    if (a.accumulate) {
#pragma unroll
      for (int c = 0; c < 4; ++c) if (c < ncols) x[c] += __bfloat162float(p[c]);
    }
    if (a.vec && ncols >= 4) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
      *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) if (c < ncols) p[c] = __float2bfloat16_rn(x[c]);
    }
  }
}
// One element of a transposed output.
__device__ __forceinline__ void put1(const Args& a, char* base, int64_t i, float v) {
  if (a.out_f32) {
    float* p = reinterpret_cast<float*>(base) + i;
    *p = a.accumulate ? *p + v : v;
  } else {
    __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(base) + i;
    *p = __float2bfloat16_rn(a.accumulate ? __bfloat162float(*p) + v : v);
  }
}

// BNT: columns of the accumulators (64, 128 or 256; a.bn <= BNT).
template <int BNT, int MODE>
__global__ void __launch_bounds__(kThreadsG, 1) k_grouped(const __grid_constant__ CUtensorMap mapA,
                                                         const __grid_constant__ CUtensorMap mapB,
                                                         const __grid_constant__ Args a, int* err) {
  constexpr int CPW = BNT / 2;          // columns of an epilogue warp
  constexpr int SB = kABytes + BNT * kBK * 2;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int S = a.split;
  unsigned char* scratch = smem + a.stages * SB;
  // split: partial tiles of the S CTAs for this CTA's rows; else: the epilogue's staging
  const int scratch_bytes = S > 1 ? kBM * (BNT + 4) * 4 : kEpiWarps * 32 * kStagePitch;
  int32_t* bnd = reinterpret_cast<int32_t*>(scratch + scratch_bytes);
  int32_t* tile0 = bnd + a.G + 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(
      reinterpret_cast<unsigned char*>(tile0) + (((a.G + 3) * 8 + 15) & ~15) - (a.G + 3) * 4);
  uint64_t* empty = full + a.stages;
  uint64_t* tfull = empty + a.stages;   // [2]
  uint64_t* tempty = tfull + 2;         // [2]
  uint64_t* red_full = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(red_full + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kCols = 2 * BNT;        // TMEM columns: two accumulators
  const int rank = S > 1 ? static_cast<int>(blockIdx.x) % S : 0;
  const int first = static_cast<int>(blockIdx.x) / S, step = static_cast<int>(gridDim.x) / S;

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) { mbar_init(full + s, 1); mbar_init(empty + s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(tfull + b, 1); mbar_init(tempty + b, kEpiWarps); }
    const int rows = kBM / S;
    mbar_init(red_full, static_cast<uint32_t>(S * 2 * (rows >= 32 ? rows / 32 : 1)));
    mbar_init_fence();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 2) scan_groups(a.offsets, a.G, static_cast<int>(a.M), a.zero_rest != 0, bnd, tile0, lane);
  tc::tc_fence_before();
  if (S > 1) cluster_sync_all(); else __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total = MODE == 0 ? tile0[a.G + 2] * a.ntn : a.G * a.mtn * a.ntn;
  const int nbox_b = a.b_mn || MODE == 1 ? (a.bn + 63) / 64 : 1;
  const uint32_t b_bytes = a.b_mn || MODE == 1 ? static_cast<uint32_t>(nbox_b * 8192) : static_cast<uint32_t>(a.bn * 128);
  auto k_begin = [&](int nk) { return static_cast<int>(static_cast<int64_t>(nk) * rank / S); };
  auto k_end = [&](int nk) { return static_cast<int>(static_cast<int64_t>(nk) * (rank + 1) / S); };

  if (warp == 0) {
    if (lane == 0) {
      int g = 0;                        // k-steps issued (position in the ring)
      bool ok = true;
      for (int t = first; t < total && ok; t += step) {
        const Tile x = tile_of<MODE>(a, bnd, tile0, t);
        const int nba = MODE == 0 ? (x.valid + a.arows - 1) / a.arows : 2;
        const uint32_t bytes = b_bytes + (MODE == 0 ? static_cast<uint32_t>(nba * a.arows * 128) : 16384u);
        for (int k = k_begin(x.nk); k < k_end(x.nk); ++k) {
          const int s = g % a.stages;
          const uint32_t u = static_cast<uint32_t>(g / a.stages);
          if (g >= a.stages && !mbar_wait(empty + s, (u & 1u) ^ 1u, err)) { ok = false; break; }
          unsigned char* As = smem + s * SB;
          unsigned char* Bs = As + kABytes;
          mbar_expect_tx(full + s, bytes);
          if (MODE == 0) {
            for (int i = 0; i < nba; ++i)
              tma_load_2d(As + i * a.arows * 128, &mapA, k * kBK, x.m0 + i * a.arows, full + s);
            if (a.b_mn) {
              for (int j = 0; j < nbox_b; ++j) tma_load_3d(Bs + j * 8192, &mapB, x.n0 + 64 * j, k * kBK, x.seg - 1, full + s);
            } else {
              tma_load_3d(Bs, &mapB, k * kBK, x.n0, x.seg - 1, full + s);
            }
          } else {
            const int r = x.r0 + k * kBK;
            tma_load_2d(As, &mapA, x.m0, r, full + s);
            tma_load_2d(As + 8192, &mapA, x.m0 + 64, r, full + s);
            for (int j = 0; j < nbox_b; ++j) tma_load_2d(Bs + j * 8192, &mapB, x.n0 + 64 * j, r, full + s);
          }
          ++g;
        }
      }
      if (!ok)
        for (int i = (g > a.stages ? g - a.stages : 0); i < g; ++i)
          mbar_drain(full + (i % a.stages), static_cast<uint32_t>(i / a.stages) & 1u);
    }
  } else if (warp == 1) {
    const uint32_t idesc = tc::idesc_bf16(a.bn, MODE, MODE == 1 ? 1 : a.b_mn);
    int g = 0, u = 0;                   // k-steps consumed, accumulators begun
    bool ok = true;
    int last = -1;
    for (int t = first; t < total && ok; t += step) {
      const Tile x = tile_of<MODE>(a, bnd, tile0, t);
      const int kb = k_begin(x.nk), ke = k_end(x.nk);
      for (int c = kb; c < ke && ok; c += a.chunk, ++u) {
        const int b = u & 1;
        if (u >= 2) ok = __all_sync(0xffffffffu, mbar_wait(tempty + b, static_cast<uint32_t>((u >> 1) - 1) & 1u, err));
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t acc = tmem + static_cast<uint32_t>(b * BNT);
        const int cend = min(ke, c + a.chunk);
        for (int k = c; k < cend; ++k) {
          const int s = g % a.stages;
          ok = __all_sync(0xffffffffu, mbar_wait(full + s, static_cast<uint32_t>(g / a.stages) & 1u, err));
          if (!ok) break;
          unsigned char* As = smem + s * SB;
          int nkk = kBK / 16;
          if (MODE == 1) {
            const int v = x.cnt - k * kBK;           // rows of the group in this k-step
            if (v < kBK) {                           // the rest belongs to the next group: cleared
              nkk = (v + 15) / 16;
              const int lo = v * 8, hi = nkk * 128;  // 16-byte units of a box
              for (int j = 0; j < 2 + nbox_b; ++j) {
                uint4* p = reinterpret_cast<uint4*>(j < 2 ? As + j * 8192 : As + kABytes + (j - 2) * 8192);
                for (int i = lo + lane; i < hi; i += 32) p[i] = make_uint4(0u, 0u, 0u, 0u);
              }
              tc::fence_proxy_async_smem();
              __syncwarp();
            }
          }
          tc::tc_fence_after();
          if (lane == 0) {
            const uint32_t a0 = smem_u32(As), b0 = a0 + kABytes;
            for (int kk = 0; kk < nkk; ++kk) {
              const uint64_t da = MODE == 0 ? tc::sdesc(a0 + kk * 32, 16, 1024) : tc::sdesc(a0 + kk * 2048, 8192, 1024);
              const uint64_t db = (MODE == 0 && !a.b_mn) ? tc::sdesc(b0 + kk * 32, 16, 1024)
                                                         : tc::sdesc(b0 + kk * 2048, 8192, 1024);
              tc::mma_bf16(acc, da, db, idesc, (k > c || kk > 0) ? 1u : 0u);
            }
            tc::mma_commit(empty + s);
          }
          __syncwarp();
          ++g;
        }
        if (lane == 0) tc::mma_commit(tfull + b);     // on an error too: it completes once the issued MMAs have
        last = u;
      }
    }
    if (!ok && last >= 0 && lane == 0) mbar_drain(tfull + (last & 1), static_cast<uint32_t>(last >> 1) & 1u);
    __syncwarp();
  } else {
    const int q = warp & 3;             // TMEM lane quadrant
    const int col0 = ((warp - 2) >> 2) * CPW;
    const int row = q * 32 + lane;      // this thread's row of the tile
    const bool cols = col0 < a.bn;
    int u = 0;
    bool ok = true;
    for (int t = first; t < total && ok; t += step) {
      const Tile x = tile_of<MODE>(a, bnd, tile0, t);
      const int kb = k_begin(x.nk), ke = k_end(x.nk);
      float acc[CPW];
#pragma unroll
      for (int c = 0; c < CPW; ++c) acc[c] = 0.f;
      for (int c = kb; c < ke; c += a.chunk, ++u) {
        const int b = u & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(tfull + b, static_cast<uint32_t>(u >> 1) & 1u, err));
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t src = tmem + static_cast<uint32_t>(b * BNT + col0) + (static_cast<uint32_t>(q * 32) << 16);
        if (cols) {
#pragma unroll
          for (int c0 = 0; c0 < CPW; c0 += 32) {
            float v[32];
            tmem_ld32(src + c0, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c0 + i] += v[i];
          }
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty + b);
      }
      if (!ok) break;
      char* out = static_cast<char*>(a.out);
      const int es = a.out_f32 ? 4 : 2;
      if (MODE == 1) out += static_cast<int64_t>(x.seg) * a.gstride * es;
      if (S > 1) {
        const int rows = kBM / S;
        constexpr int P = BNT + 4;      // floats between rows of a partial tile
        {
          const uint32_t dst = map_rank(smem_u32(scratch) + static_cast<uint32_t>(((rank * rows + row % rows) * P + col0) * 4),
                                        static_cast<uint32_t>(row / rows));
          if (cols) {
#pragma unroll
            for (int c = 0; c < CPW; c += 4)
              if (col0 + c < a.bn) st_remote(dst + c * 4, make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]));
          }
          __syncwarp();
          if (lane == 0) {
            arrive_remote(map_rank(smem_u32(red_full), static_cast<uint32_t>(q * 32 / rows)));
            if (rows < 32) arrive_remote(map_rank(smem_u32(red_full), static_cast<uint32_t>(q * 32 / rows + 1)));
          }
          __syncwarp();
        }
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(red_full, 0, err));
        if (!ok) break;
        const float* part = reinterpret_cast<const float*>(scratch);
        const int nq = a.bn / 4;
        for (int i = static_cast<int>(threadIdx.x) - 64; i < rows * nq; i += 32 * kEpiWarps) {
          // consecutive threads take consecutive columns of a row, or rows of a transposed output
          const int r = a.transposed ? i % rows : i / nq;
          const int c = 4 * (a.transposed ? i / rows : i - r * nq);
          float4 v = *reinterpret_cast<const float4*>(part + r * P + c);
          for (int p = 1; p < S; ++p) {
            const float4 w = *reinterpret_cast<const float4*>(part + (p * rows + r) * P + c);
            v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
          }
          v.x *= a.alpha; v.y *= a.alpha; v.z *= a.alpha; v.w *= a.alpha;
          const int m = rank * rows + r, n = x.n0 + c;
          if (m >= x.valid || n >= a.ndim) continue;
          if (a.transposed) {
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < a.ndim) put1(a, out, static_cast<int64_t>(n + j) * a.ld + x.m0 + m, e[j]);
          } else {
            put4(a, out + static_cast<int64_t>(x.m0 + m) * a.ld * es, n, a.ndim - n, v);
          }
        }
      } else if (a.transposed) {
        if (cols && row < x.valid) {
#pragma unroll
          for (int c = 0; c < CPW; ++c)
            if (x.n0 + col0 + c < a.ndim)
              put1(a, out, static_cast<int64_t>(x.n0 + col0 + c) * a.ld + x.m0 + row, a.alpha * acc[c]);
        }
      } else if (cols) {
        unsigned char* st = scratch + (warp - 2) * 32 * kStagePitch;
        char* base = out + static_cast<int64_t>(x.m0 + q * 32) * a.ld * es;
        const int nrows = min(32, x.valid - q * 32);
        if (!a.out_f32 && !a.accumulate && a.vec) {
          // 32 bf16 columns at a time: 64 bytes a row, four lanes a row
#pragma unroll
          for (int c0 = 0; c0 < CPW; c0 += 32) {
            if (x.n0 + col0 + c0 < a.ndim) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const __nv_bfloat162 b2 = __floats2bfloat162_rn(a.alpha * acc[c0 + 8 * j + 2 * i], a.alpha * acc[c0 + 8 * j + 2 * i + 1]);
                  w[i] = *reinterpret_cast<const uint32_t*>(&b2);
                }
                *reinterpret_cast<uint4*>(st + lane * kStagePitch + j * 16) = make_uint4(w[0], w[1], w[2], w[3]);
              }
              __syncwarp();
              const int n = x.n0 + col0 + c0 + (lane & 3) * 8;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2);
                if (r < nrows && n < a.ndim) {
                  const uint4 v = *reinterpret_cast<const uint4*>(st + r * kStagePitch + (lane & 3) * 16);
                  __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(base + static_cast<int64_t>(r) * a.ld * 2) + n;
                  if (n + 8 <= a.ndim) {
                    *reinterpret_cast<uint4*>(p) = v;
                  } else {
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    for (int j = 0; j < a.ndim - n; ++j)
                      reinterpret_cast<uint16_t*>(p)[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
                  }
                }
              }
              __syncwarp();
            }
          }
        } else {
          // 16 fp32 columns at a time
#pragma unroll
          for (int c0 = 0; c0 < CPW; c0 += 16) {
            if (x.n0 + col0 + c0 < a.ndim) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4*>(st + lane * kStagePitch + j * 16) =
                    make_float4(a.alpha * acc[c0 + 4 * j], a.alpha * acc[c0 + 4 * j + 1], a.alpha * acc[c0 + 4 * j + 2],
                                a.alpha * acc[c0 + 4 * j + 3]);
              __syncwarp();
              const int n = x.n0 + col0 + c0 + (lane & 3) * 4;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + (lane >> 2);
                if (r < nrows && n < a.ndim)
                  put4(a, base + static_cast<int64_t>(r) * a.ld * es, n, a.ndim - n,
                       *reinterpret_cast<const float4*>(st + r * kStagePitch + (lane & 3) * 16));
              }
              __syncwarp();
            }
          }
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
  if (S > 1) cluster_sync_all();        // no CTA leaves while a peer may still send to it
}

}  // namespace gr
}  // namespace dsmz
