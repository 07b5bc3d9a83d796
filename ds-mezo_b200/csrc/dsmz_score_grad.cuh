// Contrastive scoring loss with its gradient in the logits:
//   loss = sum_i a_i / n_i sum_{t in sequence i} nll_t,   nll_t = log sum_c exp(x_tc) - x_t,target
//   d loss / d x_tc = a_i / n_i (exp(x_tc) / sum_c exp(x_tc) - [c = target_t])
// (ds_mezo/controller.py:14-15, 194-201 for the loss; the reference takes no gradient of it).
//
// A row belongs to a cluster of 1 to 8 CTAs, each with a slice of the vocabulary. Pass one
// over the slice keeps a running maximum and sum of exponentials a thread; the CTAs exchange
// (max, sum) through distributed shared memory; pass two reads the slice again, from L2 (a
// cluster's barrier empties L1), and writes the gradient. HBM sees each logit once in and each
// gradient once out, which is the floor: 190 us for 2048 rows of 152064 bf16 logits, of which
// this takes 260 (0.73). The unit that makes exponentials and packs bf16 pairs is busy two
// thirds of the time (2.5 operations a logit), the rest is the latency between a slice's two
// passes. A variant that streamed whole rows through a shared-memory ring, one CTA a row, took
// 244 us there but 119 against 113 for 2048 rows of 65536; it did not stay. A short call (8
// rows of 32000) is the launches' latency: 10 us on the device with the sum's kernel launched
// beside the rows'.
// Rows need not be aligned: a slice has a scalar head up to the first 16-byte boundary,
// 16-byte accesses, and a scalar tail. The target's logit is read before the exchange, so
// the gradient may overwrite the logits.
//
// The maximum is subtracted before the scaling by log2 e: with the product first (one FMA a
// logit less) masks at the type's lowest value overflow, and logits past 2^24 lose the
// difference itself. Rows of -inf only, NaN and +inf follow the formula: NaN. A target outside
// the vocabulary makes the loss and its row of the gradient NaN.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include <type_traits>

#include "dsmz_pairs.cuh"
#include "dsmz_ptx.cuh"

namespace dsmz {
namespace sg {

constexpr int kMaxSeqs = 128;
// Largest slice of a row. 2048 rows of 152064 bf16 logits (304 KB) took 311, 297, 273 and 345 us
// with 1, 2, 4 and 8 CTAs of 256 threads a row (293, 279, 361 and 515 us with 512 threads),
// before the packed arithmetic below: more CTAs cut the tail of the last wave, and below
// slices of 76 KB their barriers cost more.
constexpr int kSliceBytes = 80 * 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct Seqs {
  int32_t n, pad;
  int64_t start[kMaxSeqs + 1];           // token rows of sequence i: [start[i], start[i+1])
  double w[kMaxSeqs];                    // a_i / n_i
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
// Not the .aligned forms: warps arrive from divergent code.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// 8-byte store to the same shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ void st_cluster(void* local, uint32_t rank, float a, float b) {
  uint32_t addr;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a), "f"(b) : "memory");
}

__device__ __forceinline__ float exp_of(float d) { return ex2(d * kLog2e); }   // d <= 0

// (m, s) <- the pair for both sets: m the larger maximum, s relative to it. An empty set is
// (-inf, 0).
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float t = fmaxf(m, m2);
  if (t == -INFINITY) { s += s2; return; }          // -inf logits alone, or NaN: s carries the NaN
  s = s * exp_of(m - t) + s2 * exp_of(m2 - t);
  m = t;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void load(const float* p, float (&x)[4]) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
  }
  __device__ static void store(float* p, const float (&x)[4]) {
    __stcs(reinterpret_cast<float4*>(p), make_float4(x[0], x[1], x[2], x[3]));
  }
  __device__ static float one(const float* p) { return *p; }
  __device__ static void put(float* p, float x) { *p = x; }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void load(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = __uint_as_float(w[q] << 16);
      x[2 * q + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
    }
  }
  __device__ static void store(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * q], x[2 * q + 1]);
      w[q] = *reinterpret_cast<const uint32_t*>(&b);
    }
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
  }
  __device__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
};

__device__ __forceinline__ F2 exp2_of(F2 a) {
  float x, y;
  a.split(x, y);
  return F2(ex2(x), ex2(y));
}
// One 16-byte vector as pairs.
__device__ __forceinline__ void load_pairs(const float* p, F2 (&x)[2], float& top) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  top = fmaxf(top, fmaxf(fmaxf(u.x, u.y), fmaxf(u.z, u.w)));
  x[0] = F2(u.x, u.y);
  x[1] = F2(u.z, u.w);
}
__device__ __forceinline__ void load_pairs(const __nv_bfloat16* p, F2 (&x)[4], float& top) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float a = __uint_as_float(w[q] << 16), b = __uint_as_float(w[q] & 0xFFFF0000u);
    top = fmaxf(top, fmaxf(a, b));
    x[q] = F2(a, b);
  }
}

// The packed instructions (273 -> 260 us) leave registers for a fifth CTA an SM.
// grid: ntok * cluster size; row = blockIdx.x / cluster size.
template <typename T>
__global__ void __launch_bounds__(256, 5) k_loss_grad(const T* logits, int64_t ld, int64_t V,
                                                   const int32_t* __restrict__ targets, Seqs seqs, double grad_scale,
                                                   T* grad, int64_t ld_grad, double* __restrict__ term) {
  constexpr int N = Vec<T>::N;
  __shared__ float2 red[8];
  __shared__ float2 part[8];                          // (max, sum) of every CTA of the cluster
  launch_dependents();                                // the sum's launch overlaps the rows
  const int tid = threadIdx.x, nt = blockDim.x;
  const uint32_t C = cluster_size(), rank = cluster_rank();
  // Another CTA's shared memory may be written once that CTA is known to run: every thread says
  // so here, and the wait comes after pass one, which hides it.
  if (C > 1) cluster_arrive_relaxed();
  const int64_t row = blockIdx.x / C;
  int si = 0;                                         // the row's sequence
  while (si + 1 < seqs.n && seqs.start[si + 1] <= row) ++si;
  const double w = seqs.w[si];
  const T* x = logits + row * ld;
  T* g = grad + row * ld_grad;
  const int32_t target = targets[row];
  const bool valid = target >= 0 && target < V;

  // this CTA's columns [c0, c1); [v0, v1) of them are whole 16-byte vectors
  const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T);   // to the row's first boundary
  const int64_t per = ((V + C - 1) / C + N - 1) / N * N;
  auto cut = [&](int64_t r) {                         // slices meet at 16-byte boundaries
    const int64_t c = r == 0 ? 0 : head + r * per;
    return c < V ? (r == C ? V : c) : V;
  };
  const int64_t c0 = cut(rank), c1 = cut(rank + 1);
  const int64_t v0 = rank == 0 ? (head < c1 ? head : c1) : c0;
  const int64_t nvec = (c1 - v0) / N, v1 = v0 + nvec * N;
  const bool same = (reinterpret_cast<uintptr_t>(g + v0) & 15) == 0;   // the gradient's row has the same phase

  const float xt = (tid == 0 && valid) ? Vec<T>::one(x + target) : 0.f;
  float m = -INFINITY, s = 0.f;
  const T* xv = x + v0;
  const int nv = static_cast<int>(nvec);
  // UN vectors a thread: one maximum and one rescaling of the running sum for all of them
  auto block = [&](auto un, int i) {
    constexpr int UN = decltype(un)::value;
    F2 y[UN][N / 2];
    float t = m;
#pragma unroll
    for (int u = 0; u < UN; ++u) load_pairs(xv + static_cast<int64_t>(i + u * nt) * N, y[u], t);
    const float b = t == -INFINITY ? 0.f : t;         // -inf logits alone: every exponential is 0
    const F2 nb(-b, -b), le(kLog2e, kLog2e);
    F2 acc(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int k = 0; k < N / 2; ++k) acc = acc + exp2_of((y[u][k] + nb) * le);
    float a0, a1;
    acc.split(a0, a1);
    s = s * exp_of(m - b) + (a0 + a1);
    m = t;
  };
  int i = tid;
  for (; i + 3 * nt < nv; i += 4 * nt) block(std::integral_constant<int, 4>{}, i);
  for (; i < nv; i += nt) block(std::integral_constant<int, 1>{}, i);
  if (tid < 2 * N) {                                  // head and tail, one element a thread
    const int64_t c = tid < N ? c0 + tid : v1 + (tid - N);
    if (c < (tid < N ? v0 : c1)) {
      const float y = Vec<T>::one(x + c);
      merge(m, s, y, y == -INFINITY ? 0.f : (y == y ? 1.f : y));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if ((tid & 31) == 0) red[tid >> 5] = make_float2(m, s);
  __syncthreads();
  // every warp merges the warps' pairs, then the CTAs' (lanes past them hold the empty pair)
  const int lane = tid & 31;
  m = lane < nt / 32 ? red[lane].x : -INFINITY;
  s = lane < nt / 32 ? red[lane].y : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if (C > 1) {
    cluster_wait();                                   // every CTA of the cluster has started
    if (tid < static_cast<int>(C)) st_cluster(&part[rank], tid, m, s);
    cluster_arrive();
    cluster_wait();                                   // and has written its pair here
    m = lane < static_cast<int>(C) ? part[lane].x : -INFINITY;
    s = lane < static_cast<int>(C) ? part[lane].y : 0.f;
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    m = __shfl_sync(0xffffffffu, m, 0);
    s = __shfl_sync(0xffffffffu, s, 0);
  }
  const float bad = __int_as_float(0x7fc00000);
  if (rank == 0 && tid == 0) {
    // the difference first: at the type's lowest value even fp64 would swallow log s
    const double nll = (static_cast<double>(m) - static_cast<double>(xt)) + log(static_cast<double>(s));
    term[row] = valid ? nll * w : static_cast<double>(bad);
  }
  const float wf = valid ? static_cast<float>(w * grad_scale) : bad;
  const float inv = 1.f / s;
  auto value = [&](float y) { return wf * (exp_of(y - m) * inv); };
  T* gv = g + v0;
  if (same) {
    auto pass = [&](auto un, int i) {
      constexpr int UN = decltype(un)::value;
      F2 y[UN][N / 2];
      float unused = 0.f;
#pragma unroll
      for (int u = 0; u < UN; ++u) load_pairs(xv + static_cast<int64_t>(i + u * nt) * N, y[u], unused);
      const F2 nm(-m, -m), le(kLog2e, kLog2e), ww(wf * inv, wf * inv);
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        float z[N];
#pragma unroll
        for (int k = 0; k < N / 2; ++k) (exp2_of((y[u][k] + nm) * le) * ww).split(z[2 * k], z[2 * k + 1]);
        Vec<T>::store(gv + static_cast<int64_t>(i + u * nt) * N, z);
      }
    };
    i = tid;
    for (; i + 3 * nt < nv; i += 4 * nt) pass(std::integral_constant<int, 4>{}, i);
    for (; i < nv; i += nt) pass(std::integral_constant<int, 1>{}, i);
  } else {
    for (i = tid; i < nv; i += nt) {
      float y[N];
      Vec<T>::load(xv + static_cast<int64_t>(i) * N, y);
#pragma unroll
      for (int k = 0; k < N; ++k) Vec<T>::put(gv + static_cast<int64_t>(i) * N + k, value(y[k]));
    }
  }
  if (tid < 2 * N) {
    const int64_t c = tid < N ? c0 + tid : v1 + (tid - N);
    if (c < (tid < N ? v0 : c1)) Vec<T>::put(g + c, value(Vec<T>::one(x + c)));
  }
  __syncthreads();                                    // the target's element, once the slice is written
  // xt was read before the first barrier, so before any gradient was written
  if (tid == 0 && valid && target >= c0 && target < c1) Vec<T>::put(g + target, wf * (exp_of(xt - m) * inv - 1.f));
}

// loss[0] = the terms' sum in fp64 in token order (each thread a contiguous run, the runs in
// thread order), rounded once.
__global__ void __launch_bounds__(256) k_loss_sum(const double* __restrict__ term, int64_t ntok, float* loss) {
  __shared__ double part[256];
  const int tid = threadIdx.x;
  grid_dependency_wait();
  const int64_t per = (ntok + 255) / 256;
  double a = 0.0;
  for (int64_t i = tid * per; i < min(ntok, (tid + 1) * per); ++i) a += term[i];
  part[tid] = a;
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int i = 0; i < 256; ++i) s += part[i];
    loss[0] = static_cast<float>(s);
  }
}

}  // namespace sg
}  // namespace dsmz
