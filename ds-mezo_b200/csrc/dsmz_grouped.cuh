// Matrix products grouped by adapter copy with ragged rows (tcgen05, bf16 operands, fp32 sums).
//
//   MODE 0   y_i  = alpha x_i W_g(i) (+ y_i)       rows i of group g are [o_g, o_{g+1})
//   MODE 1   dW_g = alpha X_g^T dY_g (+ dW_g)      the gradient in the weights
//
// The row offsets live on the device: every CTA scans them once (clamped to the rows there
// are and made monotone, so that no offset can lead out of bounds or to two owners of a row)
// and walks its tiles in ascending order. A group may be empty; its dW is zero. In MODE 0 rows
// outside every group are left as they were, or zeroed where the caller asks.
//
// A tile is 128 x BN: MODE 0 128 rows of one group, MODE 1 128 features of the wider operand.
// Twelve warps (twenty where the epilogue sets the pace):
//   warps 0, 2   TMA producers of A and of B: 64-wide k-steps into a ring of stages (issuing a
//                copy costs its warp some 300 cycles, so one producer for both held the loop);
//                warp 2 scans the offsets first
//   warp 1       TMEM owner and MMA issuer (kind::f16, M = 128, N = BN), two accumulators
//   warps 4-     epilogue: TMEM -> registers -> shared memory -> TMA stores (whole 32-row
//                pieces of a group) or coalesced stores (its last rows, accumulation)
// A tile that reaches past its group reads the neighbour's rows: harmless in MODE 0 (each
// output row depends on its own input row; rows past the group are not stored), and cleared
// in shared memory before the last k-step's MMAs in MODE 1, where they would be summed.
//
// The tensor core's accumulator rounds towards zero: an addition of 16 products loses 2^-22.3 of the
// running sum on average (measured: 5% of a sum of one sign after 2^19 additions). For fp32 outputs
// the epilogue therefore takes the accumulator into registers every kChunk k-steps and adds the
// chunks with rounding to nearest. bf16 outputs do without up to kLong k-steps a CTA, where a sum of
// one sign has lost 2^-12 of itself (half a step is 2^-9 to 2^-8), and are summed likewise beyond.
//
// Few tiles (narrow outputs): a cluster of 2 to 8 CTAs splits the contraction; each CTA copies its
// partial tile to the CTAs that own the rows (bulk copies through distributed shared memory,
// counted on the owner's barrier), and the owner adds the partials in rank order. No atomics:
// results are the same on every run.
//
// What bounds it, on one B200 (the public call back to back, of the floor at the measured copy and
// bf16 rates):
//   8192 x 3584 x 18944, 8 groups     942 us of 664 (802 at the sustained rate): the power cap and
//                                     the empty rows of ragged last tiles
//   4001 x 64 x 18944, 32 ragged      47.6 us of 35.6: the epilogue of half-filled last tiles, 5 us
//                                     until the first tile is stored
//   4133 x 28672 x 128, 4 groups      60.6 us of 39.7: 36 tiles in clusters of 3 leave 40 SMs idle,
//                                     5 us for the sum of the partial tiles
//   4096 x 3584 x 64, 2 groups        11.7 us of 4.7; one row for each of 32 groups 11.7 us of 2.3: the
//                                     host's call (12), and on the device the chain of offsets (2 us),
//                                     14 k-steps (4), partial sums (2)
//   dW of 4096 x (18944, 64)          31.6 us of 25.2: HBM, 3 us of stores after the last k-step
// Accumulation leaves through put4, old values read beside the stores that follow them: 4001 x 64 x
// 18944 takes 263 us (bf16) and 462 us (fp32; a new fp32 output 75).
//
// Every mbarrier wait gives up after Args::wait_ns (1 s unless the caller set another limit). The CTA
// then raises a flag of its own, at which its other roles give up too; an accumulator that lacks
// products is never announced, the tiles not produced are stored as NaN, copies and MMAs in flight
// are waited for, and the device's error word is set. The word is only a record: the next launch
// starts afresh.
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
constexpr int kFirstEpi = 4;            // first epilogue warp (a multiple of 4: warp % 4 is the TMEM lane quadrant)
constexpr int kChunk = 8;               // k-steps (512 products) an accumulator takes where chunks are summed
constexpr int kLong = 512;              // k-steps of a CTA beyond which bf16 outputs are summed in chunks
constexpr int kStagePitch = 80;         // bytes of a staged 64-byte row piece (conflict-free 16-byte accesses)
constexpr int kStageBytes = 4096;       // staging of an epilogue warp: 32 rows of 128 bytes
constexpr int kABytes = kBM * kBK * 2;

// Shared memory for the partial tiles that a CTA of a split receives.
__host__ __device__ constexpr int split_bytes(int S, int bnt) { return S * ((kBM + S - 1) / S) * bnt * 4; }

struct Args {
  const int32_t* offsets;               // G + 1, device
  int32_t G, mode;
  int64_t M;                            // rows of x
  int32_t mdim, ndim, kdim;             // MODE 0: -, N, K; MODE 1: wide, narrow, -
  int32_t bn;                           // MMA N (multiple of 16) = columns of a tile
  int32_t ntn, mtn;                     // column tiles; MODE 1: feature tiles
  int32_t b_mn;                         // MODE 0: W is contiguous along N
  int32_t a_slabs, b_slabs;             // an operand read along its rows' width is mapped as slabs of 64
                                        // columns (slab, row, 64) and comes in one box
  int32_t n_inner;                      // MODE 0: concurrent tiles run along the columns, not the rows
  int32_t arows;                        // MODE 0: rows of an A box
  int32_t stages, split;
  int32_t sbuf;                         // staging pieces of an epilogue warp, 1 or 2
  int32_t chunk;                        // k-steps per accumulator
  void* out;
  int64_t ld, gstride;                  // output pitch; MODE 1: elements between groups
  int32_t transposed;                   // MODE 1: element (m, n) at n * ld + m
  int32_t out_f32, accumulate, zero_rest, vec;
  int32_t tma_out;                      // mapC is valid: whole pieces leave by TMA
  float alpha;
  uint64_t wait_ns;                     // limit of a wait; 0: nothing is loaded, so that the waits run out
};
// What is in flight when a wait gave up gets this long to land: loads and copies between CTAs take
// microseconds.
constexpr uint64_t kLandNs = 10000000;

// 32 lanes x 32 consecutive fp32 columns of TMEM into v[0..31]; complete after tmem_wait().
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
// Waits for the thread's TMEM loads (their registers pass through an empty volatile asm after it,
// so that no use of them moves before the wait).
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// Box of a 3-D tensor map into this CTA's shared memory.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// 32 rows of 128 swizzled bytes from shared memory to (x, y, z) of a 3-D tensor map.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* m, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];\n cp.async.bulk.commit_group;" ::"l"(m),
               "r"(x), "r"(y), "r"(z), "r"(smem_u32(src))
               : "memory");
}
// No store of this thread reads shared memory any more.
__device__ __forceinline__ void store_read_wait() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// At most the latest group of stores does.
__device__ __forceinline__ void store_read_wait_but_one() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
// `bytes` of this CTA's shared memory to another CTA's, counted on that CTA's barrier when they
// land. (st.async, 16 bytes a lane, took 3.3 us for a 128 x 64 tile, 6 for 128 x 128.)
__device__ __forceinline__ void copy_to_rank(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "r"(smem_u32(src)), "r"(bytes), "r"(bar)
               : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// TMA loads into this CTA's shared memory that complete on a barrier of the pair's leader (a
// shared::cluster address); no multicast.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* m, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* m, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          smem_u32(dst)),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
// Whether the phase has completed, asleep for up to `ns` until it has; arrivals come from other CTAs.
__device__ __forceinline__ bool try_cluster(uint64_t* bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, "
      "p;\n}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(ns)
      : "memory");
  return ok != 0;
}
// Waits until the phase completes: false after `a.wait_ns`, or when another role of this CTA has given
// up (`gone`, in shared memory).
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_for(const Args& a, uint64_t* bar, uint32_t parity, volatile int32_t* gone) {
  if (!CLUSTER && mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = gtimer();
  while (true) {
    if (CLUSTER ? try_cluster(bar, parity, kSuspendNs) : mbar_try_wait_sleep(bar, parity)) return true;
    if (*gone != 0) return false;
    if (gtimer() - t0 >= a.wait_ns) {
      *gone = 1;
      return false;
    }
  }
}
// For copies and MMAs in flight after a wait gave up: until they complete, kLandNs at most.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = gtimer();
  while (!mbar_try_wait(bar, parity))
    if (gtimer() - t0 > kLandNs) return;
}

// Row boundaries bnd[0..G+2] = 0, the offsets (clamped to [0, M], running maximum), M; segment
// s = rows [bnd[s], bnd[s+1]): 1..G are the groups, 0 and G+1 the rows outside them. tile0[s] =
// tiles of bm rows before segment s (0 and G+1 have none unless they are zeroed). One warp.
template <int BM>
__device__ __forceinline__ void scan_groups(const int32_t* off, int G, int M, bool rest, int32_t* bnd, int32_t* tile0,
                                            int lane) {
  int carry = 0;
  for (int i0 = 0; i0 <= G; i0 += 32) {
    const int i = i0 + lane;
    int v = i <= G ? min(max(off[i], 0), M) : M;
    const int before = __shfl_up_sync(0xffffffffu, v, 1);
    if (!__all_sync(0xffffffffu, v >= (lane == 0 ? carry : before))) {       // not ascending
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v = max(v, u);
      }
      v = max(v, carry);
    }
    if (i <= G) bnd[i + 1] = v;
    carry = __shfl_sync(0xffffffffu, v, 31);
  }
  if (lane == 0) { bnd[0] = 0; bnd[G + 2] = M; }
  __syncwarp();
  int base = 0;
  for (int s0 = 0; s0 < G + 2; s0 += 32) {
    const int s = s0 + lane;
    int n = 0;
    if (s < G + 2 && (rest || (s >= 1 && s <= G))) n = (bnd[s + 1] - bnd[s] + BM - 1) / BM;
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

// i / d for 0 <= i < 2^27 and d >= 1, with inv = 1 / d rounded: the estimate is off by one at most.
__device__ __forceinline__ int fast_div(int i, int d, float inv) {
  int q = static_cast<int>(static_cast<float>(i) * inv);
  if (static_cast<float>(i) >= 16777216.f) q = i / d;          // beyond fp32's integers
  q += (i - q * d >= d) ? 1 : 0;
  q -= (i - q * d < 0) ? 1 : 0;
  return q;
}

// Walks a CTA's tiles t, t + step, ... in ascending order; BM rows a tile (MODE 0).
template <int MODE, int BM>
struct Cursor {
  int lo;                               // MODE 0: segment of the last tile found
  float inv_ntn, inv_mtn, inv_per;
  __device__ __forceinline__ Cursor(const Args& a) : lo(0) {
    inv_ntn = 1.f / static_cast<float>(a.ntn);
    if (MODE == 1) {
      inv_mtn = 1.f / static_cast<float>(a.mtn);
      inv_per = 1.f / (static_cast<float>(a.mtn) * static_cast<float>(a.ntn));
    }
  }
  __device__ __forceinline__ Tile at(const Args& a, const int32_t* bnd, const int32_t* tile0, int t) {
    Tile x;
    if (MODE == 0) {
      while (tile0[lo + 1] * a.ntn <= t) ++lo;         // t is below the total: stops at a segment with tiles
      const int t0 = tile0[lo], nm = tile0[lo + 1] - t0, local = t - t0 * a.ntn;
      int nt, mt;
      if (a.n_inner) { mt = fast_div(local, a.ntn, inv_ntn); nt = local - mt * a.ntn; } else { nt = local / nm; mt = local - nt * nm; }
      x.seg = lo;
      x.m0 = bnd[lo] + mt * BM;
      x.n0 = nt * a.bn;
      x.valid = min(BM, bnd[lo + 1] - x.m0);
      x.r0 = x.cnt = 0;
      x.nk = (lo >= 1 && lo <= a.G) ? (a.kdim + kBK - 1) / kBK : 0;
    } else {
      const int per = a.mtn * a.ntn;
      x.seg = fast_div(t, per, inv_per);
      const int local = t - x.seg * per;
      const int nt = fast_div(local, a.mtn, inv_mtn);
      x.m0 = (local - nt * a.mtn) * kBM;
      x.n0 = nt * a.bn;
      x.valid = min(kBM, a.mdim - x.m0);
      x.r0 = bnd[x.seg + 1];
      x.cnt = bnd[x.seg + 2] - x.r0;
      x.nk = (x.cnt + kBK - 1) / kBK;
    }
    return x;
  }
};

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
// One element of a transposed output (MODE 1: fp32).
__device__ __forceinline__ void put1(const Args& a, char* base, int64_t i, float v) {
  float* p = reinterpret_cast<float*>(base) + i;
  *p = a.accumulate ? *p + v : v;
}

// The first nrows rows of a staged piece (32 rows of 128 bytes, chunk j of row r at j ^ (r & 7)), of
// which `bytes` exist: eight lanes a row. All loads first: one by one with the stores they made the
// case of 127-row groups below 61 us instead of 56.
__device__ __forceinline__ void store_rows(char* out, int64_t pitch, const unsigned char* piece, int nrows, int bytes, int lane) {
  const int j = lane & 7;
  char* o = out + 16 * j + static_cast<int64_t>(lane >> 3) * pitch;
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + (lane >> 3);
    v[i] = *reinterpret_cast<const uint4*>(piece + r * 128 + ((j ^ (r & 7)) << 4));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (4 * i + (lane >> 3) < nrows && 16 * j < bytes) *reinterpret_cast<uint4*>(o) = v[i];
    o += 4 * pitch;
  }
}

// 16 fp32 columns (from column c of the warp's, of which `left` exist) of 32 rows, a row a lane, through
// the staging to the output, four lanes a row.
__device__ __forceinline__ void put16(const Args& a, char* out, unsigned char* st, const uint32_t* v, int c, int left, int nrows,
                                      int lane) {
  if (c >= left) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(st + lane * kStagePitch + j * 16) = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  __syncwarp();
  const int n = c + (lane & 3) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    if (r < nrows && n < left)
      put4(a, out + static_cast<int64_t>(r) * a.ld * (a.out_f32 ? 4 : 2), n, left - n,
           *reinterpret_cast<const float4*>(st + r * kStagePitch + (lane & 3) * 16));
  }
  __syncwarp();
}

// Rows [r0, r1) and columns [c0, c1) of a tile that was not produced become NaN. One warp.
template <int MODE>
__device__ __noinline__ void fill_nan(const Args& a, int seg, int m0, int r0, int r1, int c0, int c1, int lane) {
  const int64_t base = MODE == 1 ? static_cast<int64_t>(seg) * a.gstride : 0;
  for (int r = r0; r < r1; ++r)
    for (int c = c0 + lane; c < c1; c += 32) {
      const int64_t m = m0 + r;
      const int64_t i = base + (a.transposed ? c * a.ld + m : m * a.ld + c);
      if (a.out_f32) static_cast<float*>(a.out)[i] = __int_as_float(0x7fc00000);
      else static_cast<__nv_bfloat16*>(a.out)[i] = __float2bfloat16_rn(__int_as_float(0x7fc00000));
    }
}

// BNT: columns of the accumulators (64, 128 or 256; a.bn <= BNT). mapC: the output (3-D, boxes
// of 32 rows x 128 bytes) where a.tma_out.
// SUM: accumulators are summed in registers (fp32 outputs; bf16 ones of long contractions). EW: epilogue warps, 8, or 16 where a tile of 256 columns
// has only a few k-steps and its epilogue sets the pace.
// PAIR (MODE 0, BNT 256): a cluster of two CTAs computes 256 x 256 tiles with cta_group::2 MMAs.
// Each loads its 128 rows of A and 128 of B's rows, so a k-step costs 32 KB a CTA instead of 48;
// the CTA of rank 0 (the leader) waits for both CTAs' loads on its barriers and issues, each CTA's
// epilogue drains its own half.
template <int BNT, int MODE, bool PAIR, bool SUM, int EW>
__global__ void __launch_bounds__(32 * (kFirstEpi + EW), 1) k_grouped(const __grid_constant__ CUtensorMap mapA,
                                                         const __grid_constant__ CUtensorMap mapB,
                                                         const __grid_constant__ CUtensorMap mapC,
                                                         const __grid_constant__ Args a, int* err) {
  // columns of an epilogue warp: half a tile (a quarter), or all of a narrow one whose rows may leave as
  // 128 bytes of bf16
  constexpr int CPW = BNT == 64 && MODE == 0 ? 64 : BNT * 4 / EW;
  constexpr int SB = kABytes + (PAIR ? BNT / 2 : BNT) * kBK * 2;
  constexpr int BM = PAIR ? 2 * kBM : kBM;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int S = BNT == 256 ? 1 : a.split, stages = a.stages;          // the widest tiles are never split
  unsigned char* scratch = smem + stages * SB;
  // split: partial tiles of the S CTAs for this CTA's rows; else: the epilogue's staging
  const int scratch_bytes = S > 1 ? split_bytes(S, BNT) : EW * kStageBytes * a.sbuf;
  int32_t* bnd = reinterpret_cast<int32_t*>(scratch + scratch_bytes);
  int32_t* tile0 = bnd + a.G + 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(
      reinterpret_cast<unsigned char*>(tile0) + (((a.G + 3) * 8 + 15) & ~15) - (a.G + 3) * 4);
  uint64_t* empty = full + stages;
  uint64_t* tfull = empty + stages;     // [2]
  uint64_t* tempty = tfull + 2;         // [2]
  uint64_t* red_full = tempty + 2;
  uint64_t* dead = red_full + 1;        // the MMAs issued before a wait gave up
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dead + 1);
  volatile int32_t* gone = reinterpret_cast<volatile int32_t*>(tmem_slot + 1);      // a wait of this CTA gave up
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kCols = 2 * BNT;        // TMEM columns: two accumulators
  const int rank = PAIR ? static_cast<int>(blockIdx.x) & 1 : (S > 1 ? static_cast<int>(blockIdx.x) % S : 0);
  const int C = PAIR ? 2 : S;           // CTAs of a cluster
  const int first = static_cast<int>(blockIdx.x) / C, step = static_cast<int>(gridDim.x) / C;

  launch_dependents();
  if (warp == 2) {
    grid_dependency_wait();
    scan_groups<BM>(a.offsets, a.G, static_cast<int>(a.M), a.zero_rest != 0, bnd, tile0, lane);
  } else if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  } else if (warp == 0 && lane == 0) {
    for (int s = 0; s < stages; ++s) { mbar_init(full + s, 2); mbar_init(empty + s, 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(tfull + b, 1); mbar_init(tempty + b, (PAIR ? 2 : 1) * EW); }
    mbar_init(red_full, 1);
    mbar_init(dead, 1);
    *gone = 0;
    mbar_init_fence();
    if (S > 1) {                        // the partial tiles of this CTA's rows, from each of the S CTAs
      const int rows = (kBM + S - 1) / S;
      mbar_expect_tx(red_full, static_cast<uint32_t>(S * min(rows, kBM - rank * rows) * ((a.bn + CPW - 1) / CPW) * CPW * 4));
    }
  } else if (warp == 3 && lane == 0) {
    prefetch_map(&mapA);
    prefetch_map(&mapB);
    if (a.tma_out) prefetch_map(&mapC);
  }
  __syncwarp();
  grid_dependency_wait();               // nothing above reads or writes global memory but the scan, after its own
  tc::tc_fence_before();
  if (C > 1) { cluster_arrive(); cluster_wait(); } else { __syncthreads(); }
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int total = MODE == 0 ? tile0[a.G + 2] * a.ntn : a.G * a.mtn * a.ntn;
  const bool b_mn = MODE == 1 || a.b_mn != 0;
  const int bnc = PAIR ? a.bn / 2 : a.bn;                     // columns of B that this CTA loads
  const int nbox_b = b_mn ? (bnc + 63) / 64 : 1;
  auto k_begin = [&](int nk) { return S == 1 ? 0 : nk * rank / S; };
  auto k_end = [&](int nk) { return S == 1 ? nk : nk * (rank + 1) / S; };

  if (warp == 0 || warp == 2) {
    // As the MMA warp below: the whole warp walks the loop, one elected lane issues.
    const bool is_a = warp == 0;
    int s = 0, n = 0;                   // stage, k-steps issued
    uint32_t ph = 1;                    // parity of the wait for an empty stage (the first round passes)
    bool ok = a.wait_ns != 0;
    Cursor<MODE, BM> cur(a);
    for (int t = first; t < total && ok; t += step) {
      const Tile y = cur.at(a, bnd, tile0, t);
      const int nk = __shfl_sync(0xffffffffu, y.nk, 0), m0 = __shfl_sync(0xffffffffu, y.m0, 0);
      const int n0 = __shfl_sync(0xffffffffu, y.n0, 0), seg = __shfl_sync(0xffffffffu, y.seg, 0);
      const int r0 = __shfl_sync(0xffffffffu, y.r0, 0), valid = __shfl_sync(0xffffffffu, y.valid, 0);
      // rows of A that this CTA loads, in boxes of arows, and those of the pair's other CTA
      const int rows_a = PAIR ? min(max(valid - kBM * rank, 0), kBM) : valid;
      const int rows_p = PAIR ? min(max(valid - kBM * (1 - rank), 0), kBM) : 0;
      const int nba = MODE == 0 ? (rows_a + a.arows - 1) / a.arows : 2;
      const int nbp = PAIR ? (rows_p + a.arows - 1) / a.arows : 0;
      // bytes that complete on the barrier: both CTAs' where a pair shares the leader's
      const uint32_t bytes = !is_a ? (b_mn ? static_cast<uint32_t>(nbox_b * 8192) : static_cast<uint32_t>(bnc * 128)) * (PAIR ? 2u : 1u)
                                   : (MODE == 0 ? static_cast<uint32_t>((nba + nbp) * a.arows * 128) : 16384u);
      const int ke = k_end(nk);
      for (int k = k_begin(nk); k < ke; ++k) {
        ok = __all_sync(0xffffffffu, wait_for(a, empty + s, ph, gone));
        if (!ok) break;
        unsigned char* dst = smem + s * SB + (is_a ? 0 : kABytes);
        uint64_t* bar = full + s;
        if (PAIR) {
          if (elect_one()) {
            if (rank == 0) mbar_expect_tx(bar, bytes);
            const uint32_t lead = map_rank(smem_u32(bar), 0);
            if (is_a) {
              for (int i = 0; i < nba; ++i)
                tma_load_2d_pair(dst + i * a.arows * 128, &mapA, k * kBK, m0 + kBM * rank + i * a.arows, lead);
            } else if (b_mn) {
              if (a.b_slabs) tma_load_4d_pair(dst, &mapB, 0, k * kBK, (n0 + bnc * rank) >> 6, seg - 1, lead);
              else for (int j = 0; j < nbox_b; ++j) tma_load_3d_pair(dst + j * 8192, &mapB, n0 + bnc * rank + 64 * j, k * kBK, seg - 1, lead);
            } else {
              tma_load_3d_pair(dst, &mapB, k * kBK, n0 + bnc * rank, seg - 1, lead);
            }
          }
        } else if (elect_one()) {
          mbar_expect_tx(bar, bytes);
          if (MODE == 0) {
            if (is_a) {
              tma_load_2d(dst, &mapA, k * kBK, m0, bar);
              for (int i = 1; i < nba; ++i) tma_load_2d(dst + i * a.arows * 128, &mapA, k * kBK, m0 + i * a.arows, bar);
            } else if (b_mn) {
              if (a.b_slabs) tma_load_4d(dst, &mapB, 0, k * kBK, n0 >> 6, seg - 1, bar);
              else for (int j = 0; j < nbox_b; ++j) tma_load_3d(dst + j * 8192, &mapB, n0 + 64 * j, k * kBK, seg - 1, bar);
            } else {
              tma_load_3d(dst, &mapB, k * kBK, n0, seg - 1, bar);
            }
          } else {
            const int r = r0 + k * kBK;
            if (is_a) {
              if (a.a_slabs) {
                tma_load_3d(dst, &mapA, 0, r, m0 >> 6, bar);
              } else {
                tma_load_2d(dst, &mapA, m0, r, bar);
                tma_load_2d(dst + 8192, &mapA, m0 + 64, r, bar);
              }
            } else if (a.b_slabs) {
              tma_load_3d(dst, &mapB, 0, r, n0 >> 6, bar);
            } else {
              for (int j = 0; j < nbox_b; ++j) tma_load_2d(dst + j * 8192, &mapB, n0 + 64 * j, r, bar);
            }
          }
        }
        ++n;
        if (++s == stages) { s = 0; ph ^= 1u; }
      }
    }
    // on an error: let the loads already issued land before the CTA can exit (a pair's complete on
    // the leader, and neither CTA leaves before the other)
    if (!ok && rank * (PAIR ? 1 : 0) == 0)
      for (int i = (n > stages ? n - stages : 0); i < n; ++i)
        drain(full + (i % stages), static_cast<uint32_t>(i / stages) & 1u);
  } else if (warp == 1 && PAIR && rank != 0) {
    // the leader issues for both
  } else if (warp == 1) {
    // The whole warp walks the loop, with every branch on a vote or a broadcast, so that stages
    // and descriptors stay in uniform registers; one elected lane issues.
    const uint32_t idesc = PAIR ? tc::idesc_bf16_pair(a.bn, b_mn ? 1 : 0) : tc::idesc_bf16(a.bn, MODE, b_mn ? 1 : 0);
    // descriptors of stage 0; addresses advance in units of 16 bytes
    const uint64_t a0 = MODE == 0 ? tc::sdesc(smem_u32(smem), 16, 1024) : tc::sdesc(smem_u32(smem), 8192, 1024);
    const uint64_t b0 = b_mn ? tc::sdesc(smem_u32(smem) + kABytes, 8192, 1024) : tc::sdesc(smem_u32(smem) + kABytes, 16, 1024);
    const uint32_t ka = MODE == 0 ? 2 : 128, kb_ = b_mn ? 128 : 2;        // a 16-wide slice of the k-step
    int s = 0, u = 0;                   // stage, accumulators begun
    uint32_t ph = 0;
    bool ok = true;
    Cursor<MODE, BM> cur(a);
    for (int t = first; t < total && ok; t += step) {
      const Tile x = cur.at(a, bnd, tile0, t);
      const int nk = __shfl_sync(0xffffffffu, x.nk, 0), cnt = __shfl_sync(0xffffffffu, x.cnt, 0);
      const int kb = k_begin(nk), ke = k_end(nk);
      for (int c = kb; c < ke && ok; c += a.chunk, ++u) {
        const int b = u & 1;
        if (u >= 2) {
          const uint32_t par = static_cast<uint32_t>((u >> 1) - 1) & 1u;
          ok = __all_sync(0xffffffffu, wait_for<PAIR>(a, tempty + b, par, gone));
        }
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t acc = tmem + static_cast<uint32_t>(b * BNT);
        const int cend = min(ke, c + a.chunk);
        for (int k = c; k < cend; ++k) {
          ok = __all_sync(0xffffffffu, wait_for(a, full + s, ph, gone));
          if (!ok) break;
          const uint64_t da = a0 + static_cast<uint32_t>(s * (SB >> 4)), db = b0 + static_cast<uint32_t>(s * (SB >> 4));
          const uint32_t more = k > c ? 1u : 0u;
          int nkk = kBK / 16;
          if (MODE == 1 && cnt - k * kBK < kBK) {
            // the group ends inside this k-step: its last 16-row slice is filled up with zeros
            const int v = cnt - k * kBK;
            nkk = (v + 15) / 16;
            for (int j = 0; j < 2 + nbox_b; ++j) {
              uint4* p = reinterpret_cast<uint4*>(smem + s * SB + (j < 2 ? j * 8192 : kABytes + (j - 2) * 8192));
              for (int i = v * 8 + lane; i < nkk * 128; i += 32) p[i] = make_uint4(0u, 0u, 0u, 0u);
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
          }
          tc::tc_fence_after();
          if (PAIR) {
            if (elect_one()) {
              tc::mma_bf16_pair(acc, da, db, idesc, more);
#pragma unroll
              for (int kk = 1; kk < kBK / 16; ++kk) tc::mma_bf16_pair(acc, da + kk * ka, db + kk * kb_, idesc, 1u);
              tc::mma_commit_pair(empty + s);
            }
          } else if (elect_one()) {
            tc::mma_bf16(acc, da, db, idesc, more);
#pragma unroll
            for (int kk = 1; kk < kBK / 16; ++kk)
              if (MODE == 0 || kk < nkk) tc::mma_bf16(acc, da + kk * ka, db + kk * kb_, idesc, 1u);
            tc::mma_commit(empty + s);
          }
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;                                // an accumulator that lacks products is not announced
        if (elect_one()) {
          if (PAIR) tc::mma_commit_pair(tfull + b); else tc::mma_commit(tfull + b);
        }
      }
    }
    if (!ok) {                                         // let the MMAs already issued end
      if (elect_one()) {
        if (PAIR) tc::mma_commit_pair(dead, 1); else tc::mma_commit(dead);
      }
      drain(dead, 0);
    }
  } else if (warp >= kFirstEpi) {
    const int q = warp & 3;             // TMEM lane quadrant
    const int col0 = ((warp - kFirstEpi) >> 2) * CPW;
    const int row = q * 32 + lane;      // this thread's row of the tile
    const bool cols = col0 < a.bn;
    unsigned char* st = scratch + (warp - kFirstEpi) * a.sbuf * kStageBytes;
    const int es = a.out_f32 ? 4 : 2;
    const float alpha = a.alpha;
    const bool rows16 = a.vec && !a.accumulate && a.ndim % (16 / es) == 0;         // rows of whole 16-byte chunks
    // This warp has read accumulator b.
    auto release = [&](int b) {
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) arrive_remote(map_rank(smem_u32(tempty + b), 0)); else mbar_arrive(tempty + b);
      }
    };
    int u = 0, slot = 0;
    bool ok = true;
    int t = first;
    Cursor<MODE, BM> cur(a);
    for (; t < total; t += step) {
      Tile x = cur.at(a, bnd, tile0, t);
      if (PAIR) {                       // this CTA's half of the rows
        x.m0 += kBM * rank;
        x.valid = min(max(x.valid - kBM * rank, 0), kBM);
      }
      const int kb = k_begin(x.nk), ke = k_end(x.nk);
      const int nrows = min(32, x.valid - q * 32);             // this warp's rows that exist
      if (!SUM && S == 1) {
        // One accumulator a tile: it goes from TMEM to the output in pieces of 32 rows x 64 columns,
        // so that few registers are live. All of a warp's columns at once needed more than 168;
        // the spilled ones go to L2, since shared memory takes nearly all of L1 (4064 x 64 x 18944
        // in 32 groups of 127 rows: 61 us, 47 so).
        const bool some = x.nk > 0;                            // else the rows outside the groups: zeros
        const int b = u & 1;
        if (some) {
          ok = __all_sync(0xffffffffu, wait_for(a, tfull + b, static_cast<uint32_t>(u >> 1) & 1u, gone));
          if (!ok) break;
          tc::tc_fence_after();
        }
        const int left = a.ndim - x.n0 - col0;                 // columns from this warp's first
        const int np = cols && nrows > 0 && left > 0 ? min(CPW / 64, (left + 63) / 64) : 0;
        const uint32_t src = tmem + static_cast<uint32_t>(b * BNT + col0) + (static_cast<uint32_t>(q * 32) << 16);
        char* out = static_cast<char*>(a.out) + (static_cast<int64_t>(x.m0 + q * 32) * a.ld + x.n0 + col0) * 2;
#pragma unroll 1
        for (int p = 0; p < np; ++p) {
          // every piece commits one group of stores, so the one before the latest is this slot's
          unsigned char* piece = st + slot * kStageBytes;
          if (lane == 0) { if (a.sbuf > 1) store_read_wait_but_one(); else store_read_wait(); }
          slot = a.sbuf > 1 ? slot ^ 1 : 0;
          __syncwarp();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
            if (some) {
              tmem_ld32(src + 64 * p + 32 * h, v);
              tmem_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                asm volatile("" : "+r"(v[i]));
                v[i] = __float_as_uint(alpha * __uint_as_float(v[i]));
              }
            }
            if (rows16) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const __nv_bfloat162 b2 = __floats2bfloat162_rn(__uint_as_float(v[8 * j + 2 * i]), __uint_as_float(v[8 * j + 2 * i + 1]));
                  w[i] = *reinterpret_cast<const uint32_t*>(&b2);
                }
                *reinterpret_cast<uint4*>(piece + lane * 128 + (((4 * h + j) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
#pragma unroll
              for (int c = 0; c < 32; c += 16)
                put16(a, out, piece, v + c, 64 * p + 32 * h + c, left, nrows, lane);
            }
          }
          if (some && p + 1 == np) release(b);
          if (rows16) {
            const bool whole = a.tma_out && nrows == 32;
            if (whole) tc::fence_proxy_async_smem();
            __syncwarp();
            if (!whole) store_rows(out + 128 * p, a.ld * 2, piece, nrows, (left - 64 * p) * 2, lane);
            else if (lane == 0) tma_store_3d(&mapC, piece, x.n0 + col0 + 64 * p, x.m0 + q * 32, 0);
            if (!whole && lane == 0) store_commit();
          }
        }
        if (some) {
          if (np == 0) release(b);
          ++u;
        }
        continue;
      }
      float acc[CPW];
      if (kb >= ke) {
#pragma unroll
        for (int c = 0; c < CPW; ++c) acc[c] = 0.f;
      }
      for (int c = kb; c < ke; c += a.chunk, ++u) {
        const int b = u & 1;
        ok = __all_sync(0xffffffffu, wait_for(a, tfull + b, static_cast<uint32_t>(u >> 1) & 1u, gone));
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t src = tmem + static_cast<uint32_t>(b * BNT + col0) + (static_cast<uint32_t>(q * 32) << 16);
        if (cols) {
          if (c == kb) {                // the first accumulator as it is: all loads, then one wait
            uint32_t v[CPW];
#pragma unroll
            for (int c0 = 0; c0 < CPW; c0 += 32) tmem_ld32(src + c0, v + c0);
            tmem_wait();
#pragma unroll
            for (int i = 0; i < CPW; ++i) { asm volatile("" : "+r"(v[i])); acc[i] = __uint_as_float(v[i]); }
          } else {
#pragma unroll
            for (int c0 = 0; c0 < CPW; c0 += 16) {
              uint32_t v[16];
              tmem_ld16(src + c0, v);
              tmem_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) { asm volatile("" : "+r"(v[i])); acc[c0 + i] += __uint_as_float(v[i]); }
            }
          }
        }
        release(b);
      }
      if (S == 1 && !ok) break;
      char* out = static_cast<char*>(a.out);
      if (MODE == 1) out += static_cast<int64_t>(x.seg) * a.gstride * es;
      if (a.alpha != 1.f) {
#pragma unroll
        for (int c = 0; c < CPW; ++c) acc[c] *= a.alpha;
      }
      if (S > 1) {
        // Partial tiles [sender][column half][row][CPW]; 16-byte chunk j of row r lies at j ^ (r & 7),
        // so that neither writing a row a lane nor summing a chunk a lane meets bank conflicts.
        // Each warp stages its piece where the ring was (every load of this CTA has landed and
        // every MMA is done) and copies the rows of each owner as one block.
        const int rows = (kBM + S - 1) / S, half = col0 / CPW;
        constexpr int RB = CPW * 4, H = BNT / CPW;       // bytes of a staged row, column halves
        if (cols && ok) {
          unsigned char* mine = smem + ((warp - kFirstEpi) >> 2) * (kBM * RB) + row * RB;
#pragma unroll
          for (int c = 0; c < CPW; c += 4)
            *reinterpret_cast<float4*>(mine + (((c >> 2) ^ (row & 7)) << 4)) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
          tc::fence_proxy_async_smem();
        }
        __syncwarp();
        if (cols && ok && lane == 0) {
          int r = q * 32;
          while (r < q * 32 + 32) {
            const int to = r / rows, upto = min(min(q * 32 + 32, (to + 1) * rows), kBM);
            const uint32_t dst = smem_u32(scratch) + static_cast<uint32_t>(((rank * H + half) * rows + r - to * rows) * RB);
            copy_to_rank(map_rank(dst, static_cast<uint32_t>(to)), smem + half * (kBM * RB) + r * RB,
                         static_cast<uint32_t>((upto - r) * RB), map_rank(smem_u32(red_full), static_cast<uint32_t>(to)));
            r = upto;
          }
        }
        if (ok) ok = __all_sync(0xffffffffu, wait_for<true>(a, red_full, 0, gone));
        const int first_row = rank * rows, nr = min(rows, kBM - first_row);     // the rows this CTA owns
        constexpr int NQ = BNT / 4;
        for (int i = static_cast<int>(threadIdx.x) - 32 * kFirstEpi; i < rows * NQ; i += 32 * EW) {
          // consecutive threads take consecutive columns of a row, or rows of a transposed output
          const int r = a.transposed ? i % rows : i / NQ;
          const int c = 4 * (a.transposed ? i / rows : i % NQ);
          const int m = first_row + r, n = x.n0 + c;
          if (r >= nr || m >= x.valid || c >= a.bn || n >= a.ndim) continue;
          const unsigned char* part = scratch + ((c / CPW) * rows + r) * RB + ((((c % CPW) >> 2) ^ (m & 7)) << 4);
          float4 v = *reinterpret_cast<const float4*>(part);
          if (!ok) v.x = v.y = v.z = v.w = __int_as_float(0x7fc00000);     // a partial tile is missing
          for (int p = 1; p < S; ++p) {
            const float4 w = *reinterpret_cast<const float4*>(part + p * H * rows * RB);
            v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
          }
          if (a.transposed) {
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (n + j < a.ndim) put1(a, out, static_cast<int64_t>(n + j) * a.ld + x.m0 + m, e[j]);
          } else {
            put4(a, out + static_cast<int64_t>(x.m0 + m) * a.ld * es, n, a.ndim - n, v);
          }
        }
      } else if (!cols || nrows <= 0) {
        // nothing of this warp's piece exists
      } else if (MODE == 1 && a.transposed) {
        // a lane a feature: each column's 32 values are contiguous
        if (row < x.valid) {
          float* p = reinterpret_cast<float*>(out) + static_cast<int64_t>(x.n0 + col0) * a.ld + x.m0 + row;
          const int nc = min(CPW, a.ndim - x.n0 - col0);
#pragma unroll
          for (int c = 0; c < CPW; ++c) {
            if (c < nc) *p = a.accumulate ? *p + acc[c] : acc[c];
            p += a.ld;
          }
        }
      } else if (rows16 && a.out_f32) {
        // fp32 pieces of 32 rows x 128 bytes as above; a.sbuf of them are staged, fenced and sent
        // together.
        const bool whole = a.tma_out && (MODE == 1 || nrows == 32);
        char* base = out + (static_cast<int64_t>(x.m0 + q * 32) * a.ld + x.n0 + col0) * 4;
        const int left = a.ndim - x.n0 - col0, np = min(CPW / 32, (left + 31) / 32);         // pieces with columns
        int from = 0;                                     // first piece of the batch
#pragma unroll
        for (int p = 0; p < CPW / 32; ++p) {
          if (p < np) {
            if (p == from) {                              // the stores before have read the staging
              if (lane == 0) store_read_wait();
              __syncwarp();
            }
            unsigned char* to = st + lane * 128 + (p - from) * kStageBytes;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<float4*>(to + ((j ^ (lane & 7)) << 4)) =
                  make_float4(acc[32 * p + 4 * j], acc[32 * p + 4 * j + 1], acc[32 * p + 4 * j + 2], acc[32 * p + 4 * j + 3]);
            if (p + 1 - from == a.sbuf || p + 1 == np) {
              if (whole) tc::fence_proxy_async_smem();
              __syncwarp();
              for (int k = from; k <= p; ++k) {
                const unsigned char* piece = st + (k - from) * kStageBytes;
                if (!whole) store_rows(base + k * 128, a.ld * 4, piece, nrows, (left - 32 * k) * 4, lane);
                else if (lane == 0) tma_store_3d(&mapC, piece, x.n0 + col0 + 32 * k, x.m0 + q * 32, MODE == 1 ? x.seg : 0);
              }
              from = p + 1;
            }
          }
        }
      } else {
        // odd pitches, accumulation, and bf16 sums of chunks
        char* base = out + (static_cast<int64_t>(x.m0 + q * 32) * a.ld + x.n0 + col0) * es;
        if (lane == 0) store_read_wait();
        __syncwarp();
#pragma unroll
        for (int c = 0; c < CPW; c += 16)
          put16(a, base, st, reinterpret_cast<const uint32_t*>(acc + c), c, a.ndim - x.n0 - col0, nrows, lane);
      }
    }
    if (lane == 0) store_wait();        // the last pieces are written before the CTA ends
    if (S == 1 && !ok) {
      __syncwarp();
      for (; t < total; t += step) {    // this warp's part of every tile it did not get
        const Tile x = cur.at(a, bnd, tile0, t);
        const int top = PAIR ? kBM * rank : 0;
        fill_nan<MODE>(a, x.seg, x.m0 + top, q * 32, min(q * 32 + 32, x.valid - top), x.n0 + col0,
                       min(x.n0 + min(col0 + CPW, a.bn), a.ndim), lane);
      }
    }
  }
  __syncwarp();
  // A CTA's sends, MMAs and arrivals at others all come before its arrival here, and no CTA leaves
  // before every CTA of the cluster has arrived, so none is reached after it left.
  if (C > 1) cluster_arrive();
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    if (!PAIR) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
  if (C > 1) cluster_wait();
  if (*gone != 0 && threadIdx.x == 0) {
    atomicExch(err, 1);
    // Every CTA of the cluster has issued all that it will: what still travels to this one lands.
    const uint64_t t0 = gtimer();
    while (gtimer() - t0 < kLandNs) __nanosleep(100000);
  }
  __syncwarp();
  if (PAIR && warp == 1)                // once both CTAs are done with the pair's accumulators
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
}

}  // namespace gr
}  // namespace dsmz
