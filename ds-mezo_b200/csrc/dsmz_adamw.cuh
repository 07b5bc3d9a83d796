// AdamW over many tensors in one launch, with fp32 or 8-bit states.
//
//   m <- b1 m + (1 - b1) g           v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// fp32 states: every operation above is one fp32 rounding, in that order.
//
// 8-bit states hold blocks of 256 elements, counted from each tensor's start, with one fp32
// scale a block: m = sign q^2 s (|q| <= 127, s = max|m| / 127^2) and sqrt(v) = q^2 s (q <=
// 255, s = max sqrt(v) / 255^2). Squared codes put the levels dense near zero: the relative
// step is 2/q and the smallest level 6e-5 (m) or 1.5e-5 (sqrt v) of the block's largest
// value, where evenly spaced codes would lose everything below 1/127. A positive v never
// takes the code 0, so a denominator never falls to eps because its block has one large
// gradient. A value takes the lower of its two codes when it lies on their border. The codes are
// those of 64-bit arithmetic: a warp forms its block in fp32 with a bound on every rounding
// made, and where a value lies within that bound of a border (a block in fifteen) forms the
// block again in fp64. All in fp64, the step of a 7B set took 1634 us: 158 instructions an
// element and 39% of the conversion unit; in fp32 923 us. A block with a NaN or an infinity gets
// a scale that makes every element of the block NaN: the whole block, not one element.
//
// One CTA takes 2048 elements of one tensor, a warp one block of 256: its lanes own elements
// 4 l .. 4 l + 3 and 128 + 4 l .. + 3, so that every access of a warp is contiguous. The pass
// is bound by HBM: 28 to 30 bytes an element with fp32 states, 12 to 18 with 8-bit ones.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "dsmezo.h"

namespace dsmz {
namespace aw {

constexpr int kBlock = 256;      // elements of one scale
constexpr int kTile = 2048;      // elements of one CTA
constexpr int kThreadsAW = 256;

struct Tensor {
  void* p;                       // parameter (state_values: fp32 m out)
  const void* g;                 // gradient
  void* m; void* v;              // fp32, or int8 / uint8 codes
  float* ms; float* vs;          // scales of the codes
  void* shadow;                  // bf16 image of the updated parameter, or NULL (state_values: fp32 v out)
  int64_t n;
};

// The step's coefficients, each rounded to fp32 once.
struct Coef {
  float decay;                   // 1 - lr wd
  float inv_root;                // 1 / sqrt(1 - b2^t)
  float step;                    // lr / (1 - b1^t)
};

// Tensors of one launch, by value: a captured launch carries them, no table is uploaded.
template <int CAP>
struct Args {
  double b1, omb1, b2, omb2;
  float eps;
  Coef c;
  const Coef* dc;                // device coefficients (a step counter on the device), or NULL: c
  const float* grad_scale;       // device scalar, or NULL
  int32_t n;
  int32_t tile0[CAP + 1];        // first CTA of each tensor
  uint8_t vec[CAP];              // every array of the tensor takes 4-element accesses
  Tensor t[CAP];
};

// t <- t + 1 and the coefficients of step t, in fp64 as the host computes them.
__global__ void k_adamw_coef(int64_t* counter, const float* lr_dev, double lr, double wd, double b1, double b2,
                             int64_t step, Coef* out) {
  double t = static_cast<double>(step);
  if (counter) {
    *counter += 1;
    t = static_cast<double>(*counter);
  }
  if (lr_dev) lr = static_cast<double>(*lr_dev);
  out->decay = static_cast<float>(1.0 - lr * wd);
  out->inv_root = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, t)));
  out->step = static_cast<float>(lr / (1.0 - pow(b1, t)));
}

// Four elements from i on (nv of them inside the tensor; the others read as zero).
template <typename T>
__device__ __forceinline__ void load4(const void* base, int64_t i, int nv, bool vec, float (&x)[4]) {
  if (sizeof(T) == 4) {
    const float* p = reinterpret_cast<const float*>(base) + i;
    if (vec && nv == 4) {
      const float4 u = *reinterpret_cast<const float4*>(p);
      x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = c < nv ? p[c] : 0.f;
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + i;
    if (vec && nv == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      x[0] = __uint_as_float(u.x << 16); x[1] = __uint_as_float(u.x & 0xFFFF0000u);
      x[2] = __uint_as_float(u.y << 16); x[3] = __uint_as_float(u.y & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = c < nv ? __uint_as_float(static_cast<uint32_t>(p[c]) << 16) : 0.f;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store4(void* base, int64_t i, int nv, bool vec, const float (&x)[4]) {
  if (sizeof(T) == 4) {
    float* p = reinterpret_cast<float*>(base) + i;
    if (vec && nv == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) if (c < nv) p[c] = x[c];
    }
  } else {
    __nv_bfloat16* p = reinterpret_cast<__nv_bfloat16*>(base) + i;
    if (vec && nv == 4) {
      const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
      uint2 u;
      u.x = *reinterpret_cast<const uint32_t*>(&a);
      u.y = *reinterpret_cast<const uint32_t*>(&b);
      *reinterpret_cast<uint2*>(p) = u;
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) if (c < nv) p[c] = __float2bfloat16_rn(x[c]);
    }
  }
}
__device__ __forceinline__ uint32_t load4b(const void* base, int64_t i, int nv, bool vec) {
  const uint8_t* p = reinterpret_cast<const uint8_t*>(base) + i;
  if (vec && nv == 4) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t u = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) if (c < nv) u |= static_cast<uint32_t>(p[c]) << (8 * c);
  return u;
}
__device__ __forceinline__ void store4b(void* base, int64_t i, int nv, bool vec, uint32_t u) {
  uint8_t* p = reinterpret_cast<uint8_t*>(base) + i;
  if (vec && nv == 4) {
    *reinterpret_cast<uint32_t*>(p) = u;
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) if (c < nv) p[c] = static_cast<uint8_t>(u >> (8 * c));
  }
}
__device__ __forceinline__ int code_i8(uint32_t u, int c) { return static_cast<int>(static_cast<int8_t>(u >> (8 * c))); }
__device__ __forceinline__ int code_u8(uint32_t u, int c) { return static_cast<int>((u >> (8 * c)) & 0xFFu); }

__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Integer 0 <= i < 2^23 as fp32 without the conversion unit.
__device__ __forceinline__ float small_float(int i) {
  return __fsub_rn(__uint_as_float(0x4B000000u | static_cast<uint32_t>(i)), 8388608.f);
}
__device__ __forceinline__ float rint_small(float x) {     // |x| < 2^22
  return __fsub_rn(__fadd_rn(x, 12582912.f), 12582912.f);
}
constexpr float kU = 0x1p-24f;   // half a step of fp32: one rounding

// Largest of the warp's non-negative doubles by their bit patterns; a NaN wins over all.
__device__ __forceinline__ double warp_top(double x) {
  unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(x));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long c = __shfl_xor_sync(0xffffffffu, b, o);
    b = c > b ? c : b;
  }
  return __longlong_as_double(static_cast<long long>(b));
}
__device__ __forceinline__ double top_of(double a, double b) {
  return static_cast<unsigned long long>(__double_as_longlong(a)) > static_cast<unsigned long long>(__double_as_longlong(b)) ? a : b;
}

template <int CAP>
__device__ __forceinline__ int tensor_of(const Args<CAP>& a, int tile) {
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.tile0[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// p1 from p and the new m, v: one rounding per operation, in the order of the formula.
__device__ __forceinline__ float new_param(float p, float m, float v, const Coef& c, float eps) {
  const float den = __fadd_rn(__fmul_rn(__fsqrt_rn(v), c.inv_root), eps);
  return __fsub_rn(__fmul_rn(p, c.decay), __fmul_rn(__fdiv_rn(m, den), c.step));
}

// A block of 8-bit states in fp64, from memory (nothing of it has been stored yet): codes
// ceil(127 sqrt(|m| / top) - 1/2) and ceil(255 sqrt(sqrt(v) / top) - 1/2), one rounding per
// operation in the order of the formulas, so that values that lie on a border by their own
// arithmetic (codes and bf16 gradients in small ratios do) are decided alike everywhere.
template <typename G>
__device__ __noinline__ void exact_block(const Tensor& t, int64_t base, int lane, double b1, double omb1, double b2,
                                         double omb2, const float* grad_scale, uint32_t (&um)[2], uint32_t (&uv)[2],
                                         float& m_scale, float& v_scale) {
  const double ms = static_cast<double>(t.ms[base / kBlock]), vs = static_cast<double>(t.vs[base / kBlock]);
  const double gs = grad_scale ? static_cast<double>(*grad_scale) : 1.0;
  const int8_t* mq = reinterpret_cast<const int8_t*>(t.m);
  const uint8_t* vq = reinterpret_cast<const uint8_t*>(t.v);
  auto at = [&](int e, double& m, double& v) {
    const int64_t i = base + 128 * (e >> 2) + 4 * lane + (e & 3);
    m = v = 0.0;
    if (i >= t.n) return;                            // past the tensor: a NaN scale must not count there
    const float gf = sizeof(G) == 4 ? reinterpret_cast<const float*>(t.g)[i]
                                    : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(t.g)[i]);
    const double g = __dmul_rn(static_cast<double>(gf), gs);
    const int qm = mq[i], qv = vq[i];
    const double root = __dmul_rn(static_cast<double>(qv * qv), vs);
    m = __dadd_rn(__dmul_rn(__dmul_rn(static_cast<double>(qm * abs(qm)), ms), b1), __dmul_rn(g, omb1));
    v = __dadd_rn(__dmul_rn(__dmul_rn(root, root), b2), __dmul_rn(__dmul_rn(g, omb2), g));
  };
  double mt = 0.0, vt = 0.0;
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    double m, v;
    at(e, m, v);
    mt = top_of(mt, fabs(m));
    vt = top_of(vt, fabs(v));
  }
  mt = warp_top(mt);
  vt = warp_top(vt);
  const double rt = __dsqrt_rn(vt);
  um[0] = um[1] = uv[0] = uv[1] = 0;
#pragma unroll 1
  for (int e = 0; e < 8; ++e) {
    double m, v;
    at(e, m, v);
    int qm = mt > 0.0 ? static_cast<int>(ceil(__dadd_rn(__dmul_rn(127.0, __dsqrt_rn(__ddiv_rn(fabs(m), mt))), -0.5))) : 0;
    int qv = rt > 0.0 ? static_cast<int>(ceil(__dadd_rn(__dmul_rn(255.0, __dsqrt_rn(__ddiv_rn(__dsqrt_rn(v), rt))), -0.5))) : 0;
    qm = min(max(qm, 0), 127);
    qv = min(max(qv, v > 0.0 ? 1 : 0), 255);
    const uint32_t cm = (static_cast<uint32_t>(m < 0.0 ? -qm : qm) & 0xFFu) << (8 * (e & 3));
    const uint32_t cv = static_cast<uint32_t>(qv) << (8 * (e & 3));
    if (e < 4) { um[0] |= cm; uv[0] |= cv; } else { um[1] |= cm; uv[1] |= cv; }
  }
  m_scale = static_cast<float>(mt / 16129.0 + (mt - mt));      // an infinite top: a NaN scale
  v_scale = static_cast<float>(rt / 65025.0 + (rt - rt));
}

// P, G: float or __nv_bfloat16 (parameter and gradient types); BITS: 32 or 8.
template <int CAP, typename P, typename G, int BITS>
__global__ void __launch_bounds__(kThreadsAW) k_adamw(const __grid_constant__ Args<CAP> a) {
  const int ti = tensor_of(a, static_cast<int>(blockIdx.x));
  const Tensor& t = a.t[ti];
  const int lane = threadIdx.x & 31;
  const int64_t base = static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.tile0[ti]) * kTile +
                       (threadIdx.x >> 5) * kBlock;
  if (base >= t.n) return;                         // the whole warp: no element of this block exists
  const bool vec = a.vec[ti] != 0;
  int64_t i[2];
  int nv[2];
  float p[2][4], g[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    i[h] = base + 128 * h + 4 * lane;
    const int64_t left = t.n - i[h];
    nv[h] = left >= 4 ? 4 : (left > 0 ? static_cast<int>(left) : 0);
    load4<P>(t.p, i[h], nv[h], vec, p[h]);
    load4<G>(t.g, i[h], nv[h], vec, g[h]);
  }
  Coef c = a.c;
  if (a.dc) c = *a.dc;
  if (BITS == 32) {
    const float b1 = static_cast<float>(a.b1), o1 = static_cast<float>(a.omb1);
    const float b2 = static_cast<float>(a.b2), o2 = static_cast<float>(a.omb2);
    float m[2][4], v[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      load4<float>(t.m, i[h], nv[h], vec, m[h]);
      load4<float>(t.v, i[h], nv[h], vec, v[h]);
    }
    const float gs = a.grad_scale ? *a.grad_scale : 1.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float gg = a.grad_scale ? __fmul_rn(g[h][k], gs) : g[h][k];
        m[h][k] = __fadd_rn(__fmul_rn(m[h][k], b1), __fmul_rn(gg, o1));
        v[h][k] = __fadd_rn(__fmul_rn(v[h][k], b2), __fmul_rn(__fmul_rn(gg, o2), gg));
        p[h][k] = new_param(p[h][k], m[h][k], v[h][k], c, a.eps);
      }
      store4<float>(t.m, i[h], nv[h], vec, m[h]);
      store4<float>(t.v, i[h], nv[h], vec, v[h]);
    }
  } else {
    const int64_t blk = base / kBlock;
    const float ms = t.ms[blk], vs = t.vs[blk];
    uint32_t mq[2], vq[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mq[h] = load4b(t.m, i[h], nv[h], vec);
      vq[h] = load4b(t.v, i[h], nv[h], vec);
    }
    const float gs = a.grad_scale ? *a.grad_scale : 1.f;
    const float b1 = static_cast<float>(a.b1), o1 = static_cast<float>(a.omb1);
    const float b2 = static_cast<float>(a.b2), o2 = static_cast<float>(a.omb2);
    float m[2][4], v[2][4], e[2][4], root[2][4];
    uint32_t mtb = 0, vtb = 0, etb = 0, positive = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = k < nv[h];                     // past the tensor: a NaN scale must not count there
        const float gg = __fmul_rn(g[h][k], gs);
        const int qm = code_i8(mq[h], k), qv = code_u8(vq[h], k);
        const float q2 = __fmul_rn(small_float(qm * qm), ms), old = __fmul_rn(small_float(qv * qv), vs);
        const float x = __fmul_rn(qm < 0 ? -q2 : q2, b1), y = __fmul_rn(gg, o1);
        m[h][k] = in ? __fadd_rn(x, y) : 0.f;
        e[h][k] = in ? __fadd_rn(fabsf(x), fabsf(y)) : 0.f;      // |m|'s error is at most 4 kU e
        v[h][k] = in ? __fadd_rn(__fmul_rn(__fmul_rn(old, old), b2), __fmul_rn(__fmul_rn(gg, o2), gg)) : 0.f;   // 6 kU
        if ((old != 0.f && b2 != 0.f) || gg != 0.f) positive |= 1u << (4 * h + k);
        mtb = max(mtb, __float_as_uint(fabsf(m[h][k])));         // as integers: a NaN wins
        vtb = max(vtb, __float_as_uint(v[h][k]));
        etb = max(etb, __float_as_uint(e[h][k]));
        // the update itself with the one-instruction root and quotient (2 and 4 kU): its error
        // is far below that of the 8-bit states it is made from
        root[h][k] = sqrt_approx(v[h][k]);
        p[h][k] = __fsub_rn(__fmul_rn(p[h][k], c.decay),
                            __fmul_rn(__fdividef(m[h][k], fmaf(root[h][k], c.inv_root, a.eps)), c.step));
      }
    const float mt = __uint_as_float(__reduce_max_sync(0xffffffffu, mtb));
    const float vt = __uint_as_float(__reduce_max_sync(0xffffffffu, vtb));
    const float et = __uint_as_float(__reduce_max_sync(0xffffffffu, etb));
    // fp32 carries the block where its largest values are well inside the range and the means
    // do not cancel throughout; an all-zero block is exact
    const bool mok = (mt > 0x1p-90f && mt < 0x1p100f && et <= 16.f * mt) || et == 0.f;
    const bool vok = (vt > 0x1p-70f && vt < 0x1p100f) || (vt == 0.f && !__any_sync(0xffffffffu, positive != 0));
    bool near = !(mok && vok);
    const float im = mt > 0.f ? __fdividef(16129.f, mt) : 0.f, iv = vt > 0.f ? __fdividef(4228250625.f, vt) : 0.f;
    const float ir = sqrt_approx(iv);
    // error of y = |m| im: 4 kU e im from m, and relative 4 kU et / mt from the top, 4 kU from
    // the quotient, its product and the top's own
    const float ey = kU * (4.f * __fdividef(et, mt) + 6.f);
    uint32_t um[2], uv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      um[h] = uv[h] = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // the border (j + 1/2)^2 nearest to y = (127 sqrt(|m| / top))^2 splits codes j and j + 1
        const float y = fabsf(m[h][k]) * im;
        const float j = fmaxf(rint_small(sqrt_approx(y) - 0.5f), 0.f);
        const float bj = (j + 0.5f) * (j + 0.5f);                            // exact
        near |= fabsf(y - bj) <= fmaf(4.f * kU * im, e[h][k], ey * y);
        const int qm = min(static_cast<int>(__float_as_uint(j + 8388608.f) & 0xFFu) + (y > bj ? 1 : 0), 127);
        // likewise (j + 1/2)^4 and (255 sqrt(sqrt(v) / top))^4: relative 6 kU for v, 6 for the
        // top, 4 for the quotient and its product, 2 for the border
        const float z = v[h][k] * iv;
        const float jv = fmaxf(rint_small(sqrt_approx(root[h][k] * ir) - 0.5f), 0.f);
        const float b2j = (jv + 0.5f) * (jv + 0.5f), b4 = b2j * b2j;
        near |= fabsf(z - b4) <= 20.f * kU * b4;
        int qv = min(static_cast<int>(__float_as_uint(jv + 8388608.f) & 0xFFu) + (z > b4 ? 1 : 0), 255);
        if (qv == 0 && (positive >> (4 * h + k) & 1u)) qv = 1;
        um[h] |= (static_cast<uint32_t>(m[h][k] < 0.f ? -qm : qm) & 0xFFu) << (8 * k);
        uv[h] |= static_cast<uint32_t>(qv) << (8 * k);
      }
    }
    float msn = __fmul_rn(mt, 1.f / 16129.f), vsn = __fmul_rn(__fsqrt_rn(vt), 1.f / 65025.f);
    if (__any_sync(0xffffffffu, near))
      exact_block<G>(t, base, lane, a.b1, a.omb1, a.b2, a.omb2, a.grad_scale, um, uv, msn, vsn);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      store4b(t.m, i[h], nv[h], vec, um[h]);
      store4b(t.v, i[h], nv[h], vec, uv[h]);
    }
    if (lane == 0) {
      t.ms[blk] = msn;
      t.vs[blk] = vsn;
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    store4<P>(t.p, i[h], nv[h], vec, p[h]);
    if (sizeof(P) == 4 && t.shadow) store4<__nv_bfloat16>(t.shadow, i[h], nv[h], vec, p[h]);
  }
}

// The fp32 values that 8-bit codes stand for.
template <int CAP>
__global__ void __launch_bounds__(kThreadsAW) k_adamw_values(const __grid_constant__ Args<CAP> a) {
  const int ti = tensor_of(a, static_cast<int>(blockIdx.x));
  const Tensor& t = a.t[ti];
  const int lane = threadIdx.x & 31;
  const int64_t base = static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.tile0[ti]) * kTile +
                       (threadIdx.x >> 5) * kBlock;
  if (base >= t.n) return;
  const bool vec = a.vec[ti] != 0;
  const double ms = static_cast<double>(t.ms[base / kBlock]), vs = static_cast<double>(t.vs[base / kBlock]);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t i = base + 128 * h + 4 * lane;
    const int64_t left = t.n - i;
    const int nv = left >= 4 ? 4 : (left > 0 ? static_cast<int>(left) : 0);
    const uint32_t um = load4b(t.m, i, nv, vec), uv = load4b(t.v, i, nv, vec);
    float m[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int qm = code_i8(um, k), qv = code_u8(uv, k);
      const double root = static_cast<double>(qv * qv) * vs;
      m[k] = static_cast<float>(static_cast<double>(qm * abs(qm)) * ms);
      v[k] = static_cast<float>(root * root);
    }
    store4<float>(t.p, i, nv, vec, m);
    store4<float>(t.shadow, i, nv, vec, v);
  }
}

}  // namespace aw
}  // namespace dsmz
