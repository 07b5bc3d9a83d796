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
// this takes 256 (0.74). The unit that makes exponentials and packs bf16 pairs is busy two
// thirds of the time (2.5 operations a logit), the rest is the latency between a slice's two
// passes. A variant that streamed whole rows through a shared-memory ring, one CTA a row, took
// 244 us there but 119 against 113 for 2048 rows of 65536; it did not stay. A short call (8
// rows of 32000) is the launches' latency: 10 us on the device with the sum's kernel launched
// beside the rows'.
// Rows need not be aligned: a slice has a scalar head up to the first 16-byte boundary,
// 16-byte accesses, and a scalar tail. The target's logit is read before the exchange, so
// the gradient may overwrite the logits.
//
// The target is left out of maximum and sum (it counts as -inf there) and joins at the end: with
// R = sum over the others and e = exp(x_target - m),
//   d loss / d x_target = -a_i / n_i R / (R + e),   nll = log1p(R) where the target is the maximum.
// A likely token has R far below 1; a sum that holds its 1 keeps R to 6e-8 only, and p - 1 and
// log(sum) lose the rest (a tenth of both at 1 - p = 1e-6, all of them below 6e-8).
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
// The largest of t and the elements of UN 16-byte vectors, NaN aside.
template <int UN>
__device__ __forceinline__ float top_of(const uint4* raw, float t, float) {
#pragma unroll
  for (int u = 0; u < UN; ++u)
    t = fmaxf(t, fmaxf(fmaxf(__uint_as_float(raw[u].x), __uint_as_float(raw[u].y)),
                       fmaxf(__uint_as_float(raw[u].z), __uint_as_float(raw[u].w))));
  return t;
}
template <int UN>
__device__ __forceinline__ float top_of(const uint4* raw, float t, __nv_bfloat16) {
  auto pair = [](uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
  __nv_bfloat162 p = __hmax2(__hmax2(pair(raw[0].x), pair(raw[0].y)), __hmax2(pair(raw[0].z), pair(raw[0].w)));
#pragma unroll
  for (int u = 1; u < UN; ++u)
    p = __hmax2(p, __hmax2(__hmax2(pair(raw[u].x), pair(raw[u].y)), __hmax2(pair(raw[u].z), pair(raw[u].w))));
  return fmaxf(t, fmaxf(__low2float(p), __high2float(p)));
}
// Pair k of a 16-byte vector (4 floats or 8 bf16).
template <typename T>
__device__ __forceinline__ F2 pair_of(const uint4& u, int k) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if (sizeof(T) == 4) return F2(__uint_as_float(w[2 * k]), __uint_as_float(w[2 * k + 1]));
  return F2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xFFFF0000u));
}

// This CTA's columns [c0, c1) of a row at x; from v0 on they hold nv whole 16-byte vectors. Slices
// meet at 16-byte boundaries.
template <typename T>
struct Slice { int c0, c1, v0, nv; };
template <typename T>
__device__ __forceinline__ Slice<T> slice_of(const T* x, int64_t V) {
  constexpr int N = Vec<T>::N;
  const uint32_t C = cluster_size(), rank = cluster_rank();
  const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T);   // to the row's first boundary
  const int64_t per = ((V + C - 1) / C + N - 1) / N * N;
  auto cut = [&](uint32_t r) {
    const int64_t c = r == 0 ? 0 : head + r * per;
    return static_cast<int>(c < V ? (r == C ? V : c) : V);            // V < 2^31
  };
  Slice<T> s;
  s.c0 = cut(rank);
  s.c1 = cut(rank + 1);
  s.v0 = rank == 0 ? min(static_cast<int>(head), s.c1) : s.c0;
  s.nv = (s.c1 - s.v0) / N;
  return s;
}

// The packed instructions (273 -> 260 us) leave registers for a fifth CTA an SM. 48 registers are all
// there are: a vector stays as it was read until its exponentials are formed, and the largest of bf16 is
// taken two by two, or the loops spill (272 us).
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
  const T* x = logits + row * ld;
  const int32_t target = targets[row];

  __shared__ float target_logit;
  __shared__ double row_weight;
  float m = -INFINITY, s = 0.f;
  const Slice<T> sl = slice_of(x, V);
  const T* xv = x + sl.v0;
  const int nv = sl.nv;
  auto vec = [&](int i) { return *reinterpret_cast<const uint4*>(xv + static_cast<int64_t>(i) * N); };
  // UN vectors of a thread join (m, s): one maximum and one rescaling of the running sum for all of them
  auto joined = [&](auto un, const uint4* raw) {
    constexpr int UN = decltype(un)::value;
    const float t = top_of<UN>(raw, m, T());
    const float b = t == -INFINITY ? 0.f : t;         // -inf logits alone: every exponential is 0
    const F2 nb(-b, -b), le(kLog2e, kLog2e);
    F2 acc(0.f, 0.f);
#pragma unroll
    for (int u = 0; u < UN; ++u)
#pragma unroll
      for (int k = 0; k < N / 2; ++k) acc = acc + exp2_of((pair_of<T>(raw[u], k) + nb) * le);
    float a0, a1;
    acc.split(a0, a1);
    return make_float2(t, s * exp_of(m - b) + (a0 + a1));
  };
  // The first loads are under way before anything asks for the target's id.
  int i = tid;
  uint4 raw[4];
  const bool blocks = i + 3 * nt < nv;
  if (blocks) {
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = vec(i + u * nt);
  }
  const bool valid = target >= 0 && target < V;
  const float xt0 = tid == 0 && valid ? Vec<T>::one(x + target) : -INFINITY;
  // The vector that holds the target (-1: none of this slice): the loops leave it out, and its other
  // elements are taken one by one.
  const int tv = valid && target >= sl.v0 && target < sl.v0 + nv * N ? (target - sl.v0) / N : -1;
  // and the first vector of this thread's block with it (nt is a power of two)
  const int hit = tv >= 0 && ((tv - tid) & (nt - 1)) == 0 ? tv - ((tv - tid) & (4 * nt - 1)) : -1;
  if (blocks)
    while (true) {
      if (i == hit) {
        const uint32_t none = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;              // -inf
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + u * nt == tv) raw[u] = make_uint4(none, none, none, none);
      }
      const float2 z = joined(std::integral_constant<int, 4>{}, raw);
      m = z.x;
      s = z.y;
      i += 4 * nt;
      if (i + 3 * nt >= nv) break;
#pragma unroll
      for (int u = 0; u < 4; ++u) raw[u] = vec(i + u * nt);
    }
#pragma unroll
  for (int u = 0; u < 3; ++u) raw[u] = i + u * nt < nv ? vec(i + u * nt) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int u = 0; u < 3; ++u)
    if (i + u * nt < nv && i + u * nt != tv) {
      const float2 z = joined(std::integral_constant<int, 1>{}, raw + u);
      m = z.x;
      s = z.y;
    }
  const int64_t c0 = sl.c0, c1 = sl.c1, v0 = sl.v0, v1 = v0 + static_cast<int64_t>(nv) * N;
  T* g = grad + row * ld_grad;
  const bool same = (reinterpret_cast<uintptr_t>(g + v0) & 15) == 0;   // the gradient's row has the same phase
  if (tid < (tv < 0 ? 2 : 3) * N) {                   // head, tail and target's vector, one element a thread
    int64_t c = c0 + tid, end = v0;
    if (tid >= N) c = v1 + (tid - N), end = c1;
    if (tid >= 2 * N) c = v0 + static_cast<int64_t>(tv) * N + (tid - 2 * N), end = v1;
    if (c < end && (c != target || !valid)) {
      const float y = Vec<T>::one(x + c);
      merge(m, s, y, y == -INFINITY ? 0.f : (y == y ? 1.f : y));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if ((tid & 31) == 0) red[tid >> 5] = make_float2(m, s);
  if (tid == 0) {
    target_logit = xt0;
    int si = 0;                                       // the row's sequence
    while (si + 1 < seqs.n && seqs.start[si + 1] <= row) ++si;
    row_weight = seqs.w[si];
  }
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
  // the target joins: s = rest + its exponential
  const float xt = target_logit, top = fmaxf(m, xt);
  const float rest = m == -INFINITY ? s : s * exp_of(m - top);          // nothing but the target: 0, or a NaN
  s = rest + exp_of(xt - top);
  m = top;
  const double w = row_weight;
  const float bad = __int_as_float(0x7fc00000);
  if (rank == 0 && tid == 0) {
    // the difference first: at the type's lowest value even fp64 would swallow log s
    const double nll = m == xt && s == s ? log1p(static_cast<double>(rest))
                                         : (static_cast<double>(m) - static_cast<double>(xt)) + log(static_cast<double>(s));
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
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const uint4 q = vec(i + u * nt);
#pragma unroll
        for (int k = 0; k < N / 2; ++k) y[u][k] = pair_of<T>(q, k);
      }
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
  if (tid == 0 && valid && target >= c0 && target < c1) Vec<T>::put(g + target, -wf * (rest / s));
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
