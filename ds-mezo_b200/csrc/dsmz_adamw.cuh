// AdamW over many tensors, up to 256 in one launch, with fp32 or 8-bit states.
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
// made, decides the elements that lie within that bound of a border (one block in thirty has
// one) in fp64, and takes the scales from the one or two elements that can be the largest,
// formed again in fp64. A 7B set (161.5 M elements; bf16 gradients and shadow, 16 bytes an
// element, 394 us at the measured copy rate) took 1634 us with everything in fp64, 1376 in
// fp32 with blocks near a border done again whole, 723 with single elements done again, no
// conversions and a path without bounds for whole blocks, 608 with packed arithmetic, 576 in
// CTAs of two warps. What bounds it is instruction issue and latency: 84 instructions an
// element, 32 warps an SM of 64 registers, out of which a thread spills 64 to 72 bytes (116 to 136
// read back) for its eight elements.
// A block with a NaN or an infinity gets a scale that makes every element of the block NaN: the
// whole block, not one element.
//
// One CTA takes a tile of one tensor, a warp one block of 256: its lanes own elements
// 4 l .. 4 l + 3 and 128 + 4 l .. + 3, so that every access of a warp is contiguous. With fp32
// states (28 to 30 bytes an element) HBM bounds the pass: 731 us for the same 7B set, 739 at
// the measured copy rate.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "dsmezo.h"
#include "dsmz_pairs.cuh"

namespace dsmz {
namespace aw {

constexpr int kBlock = 256;      // elements of one scale
// Small CTAs start and end apart from each other, so that the loads of some fall into the
// arithmetic of others: 608, 583 and 576 us for the 8-bit step with 256, 128 and 64 threads, 32 warps an
// SM of 64 registers each (28 of 72: 624, 24 of 80: 663, 36 of 56: 635). fp32 states: 715 and 713.
constexpr int kThreadsAW = 64;
constexpr int kTile = 8 * kThreadsAW;   // elements of one CTA

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
  double b1, omb1, b2, omb2;     // 1 - b formed in fp64
  float fb1, fo1, fb2, fo2;      // the same rounded once
  float eps;
  Coef c;
  const Coef* dc;                // device coefficients (a step counter on the device), or NULL: c
  const float* grad_scale;       // device scalar, or NULL
  int32_t n;
  int32_t tiles;                 // kTile-element tiles of one CTA
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

__device__ __forceinline__ float sqrt_ftz(float x) {        // relative error 2^-23; below 2^-126: 0
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_ftz(float x) {         // relative error 2^-23
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The low bytes of four words in one.
__device__ __forceinline__ uint32_t pack4(const uint32_t (&c)[4]) {
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
// 2^23 + byte k of u, without the conversion unit.
__device__ __forceinline__ float byte_float(uint32_t u, int k) {
  return __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440u + static_cast<uint32_t>(k)));
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

// New m and v of one element of 8-bit states in fp64, one rounding per operation.
__device__ __forceinline__ double mean64(int q, float scale, float g, double gs, double b1, double omb1) {
  return __dadd_rn(__dmul_rn(__dmul_rn(static_cast<double>(q * abs(q)), static_cast<double>(scale)), b1),
                   __dmul_rn(__dmul_rn(static_cast<double>(g), gs), omb1));
}
__device__ __forceinline__ double root64(int q, float scale, float g, double gs, double b2, double omb2) {
  const double root = __dmul_rn(static_cast<double>(q * q), static_cast<double>(scale));
  const double gg = __dmul_rn(static_cast<double>(g), gs);
  return __dadd_rn(__dmul_rn(__dmul_rn(root, root), b2), __dmul_rn(__dmul_rn(gg, omb2), gg));
}

// Codes in fp64, one rounding per operation in the order of the formulas, so that values that
// lie on a border by their own arithmetic (codes and bf16 gradients in small ratios do) are
// decided alike everywhere: ceil(127 sqrt(|m| / top) - 1/2) and, with root_top = sqrt(top v),
// ceil(255 sqrt(sqrt(v) / root_top) - 1/2).
__device__ __forceinline__ int mean_code(double a, double top) {
  const int q = top > 0.0 ? static_cast<int>(ceil(__dadd_rn(__dmul_rn(127.0, __dsqrt_rn(__ddiv_rn(a, top))), -0.5))) : 0;
  return min(max(q, 0), 127);
}
__device__ __forceinline__ int root_code(double v, double root_top) {
  const int q = root_top > 0.0
                    ? static_cast<int>(ceil(__dadd_rn(__dmul_rn(255.0, __dsqrt_rn(__ddiv_rn(__dsqrt_rn(v), root_top))), -0.5)))
                    : 0;
  return min(max(q, v > 0.0 ? 1 : 0), 255);
}

// A block of 8-bit states in fp64, from memory (nothing of it has been stored yet): blocks
// outside fp32's range, with NaN or infinities, or whose means cancel throughout.
template <typename G>
__device__ __noinline__ void exact_block(const Tensor& t, int64_t base, int lane, double b1, double omb1, double b2,
                                         double omb2, const float* grad_scale, uint32_t (&um)[2], uint32_t (&uv)[2],
                                         float& m_scale, float& v_scale) {
  const float ms = t.ms[base / kBlock], vs = t.vs[base / kBlock];
  const double gs = grad_scale ? static_cast<double>(*grad_scale) : 1.0;
  const int8_t* mq = reinterpret_cast<const int8_t*>(t.m);
  const uint8_t* vq = reinterpret_cast<const uint8_t*>(t.v);
  auto at = [&](int e, double& m, double& v) {
    const int64_t i = base + 128 * (e >> 2) + 4 * lane + (e & 3);
    m = v = 0.0;
    if (i >= t.n) return;                            // past the tensor: a NaN scale must not count there
    const float gf = sizeof(G) == 4 ? reinterpret_cast<const float*>(t.g)[i]
                                    : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(t.g)[i]);
    m = mean64(mq[i], ms, gf, gs, b1, omb1);
    v = root64(vq[i], vs, gf, gs, b2, omb2);
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
    const int qm = mean_code(fabs(m), mt), qv = root_code(v, rt);
    const uint32_t cm = (static_cast<uint32_t>(m < 0.0 ? -qm : qm) & 0xFFu) << (8 * (e & 3));
    const uint32_t cv = static_cast<uint32_t>(qv) << (8 * (e & 3));
    if (e < 4) { um[0] |= cm; uv[0] |= cv; } else { um[1] |= cm; uv[1] |= cv; }
  }
  m_scale = static_cast<float>(mt / 16129.0 + (mt - mt));      // an infinite top: a NaN scale
  v_scale = static_cast<float>(rt / 65025.0 + (rt - rt));
}

// P, G: float or __nv_bfloat16 (parameter and gradient types); BITS: 32 or 8.
// FULL: the block lies inside the tensor and every array takes 4-element accesses.
template <int CAP, typename P, typename G, int BITS, bool FULL>
__device__ __forceinline__ void step_block(const Args<CAP>& a, const Tensor& t, int64_t base, int lane, bool vec_) {
  const bool vec = FULL ? true : vec_;
  int64_t i[2];
  int nv[2];
  float p[2][4], g[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    i[h] = base + 128 * h + 4 * lane;
    const int64_t left = t.n - i[h];
    nv[h] = FULL || left >= 4 ? 4 : (left > 0 ? static_cast<int>(left) : 0);
    load4<P>(t.p, i[h], nv[h], vec, p[h]);
    load4<G>(t.g, i[h], nv[h], vec, g[h]);
  }
  Coef c = a.c;
  if (a.dc) c = *a.dc;
  if (BITS == 32) {
    const float b1 = a.fb1, o1 = a.fo1, b2 = a.fb2, o2 = a.fo2;
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
      store4<P>(t.p, i[h], nv[h], vec, p[h]);
      if (sizeof(P) == 4 && t.shadow) store4<__nv_bfloat16>(t.shadow, i[h], nv[h], vec, p[h]);
    }
  } else {
    const int64_t blk = base / kBlock;
    const float ms = t.ms[blk], vs = t.vs[blk];
    uint32_t mq[2], vq[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mq[h] = load4b(t.m, i[h], nv[h], vec) ^ 0x80808080u;               // q + 128
      vq[h] = load4b(t.v, i[h], nv[h], vec);
      if (a.b2 == 0.0 || vs == 0.f) vq[h] = 0;                           // no old second moment
    }
    if (a.grad_scale) {
      const float gs = *a.grad_scale;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) g[h][k] *= gs;
    }
    const float o1 = a.fo1, o2 = a.fo2, cm = ms * a.fb1, cv = (vs * vs) * a.fb2;
    F2 m2[2][2], v2[2][2];                             // the new m and v, two elements a pair
    uint32_t mtb = 0, vtb = 0;
    float gt = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int k = 2 * j;
        const F2 gg(g[h][k], g[h][k + 1]);
        float q0, q1;
        const F2 qm = F2(byte_float(mq[h], k), byte_float(mq[h], k + 1)) + F2(-8388736.f);
        qm.split(q0, q1);
        // error of the mean: at most 3 kU of the old term, 3 kU of the new, kU of the sum
        F2 mm = fma2(gg, F2(o1), (qm * F2(fabsf(q0), fabsf(q1))) * F2(cm));
        const F2 qv = F2(byte_float(vq[h], k), byte_float(vq[h], k + 1)) + F2(-8388608.f);
        const F2 q2 = qv * qv;
        F2 vv = fma2(gg * gg, F2(o2), (q2 * q2) * F2(cv));                // 6 kU
        float a0, a1, b0, b1;
        mm.split(a0, a1);
        vv.split(b0, b1);
        if (!FULL) {                                   // past the tensor: a NaN scale must not count there
          if (k >= nv[h]) a0 = b0 = 0.f;
          if (k + 1 >= nv[h]) a1 = b1 = 0.f;
          mm = F2(a0, a1);
          vv = F2(b0, b1);
        }
        m2[h][j] = mm;
        v2[h][j] = vv;
        mtb = max(max(mtb, __float_as_uint(fabsf(a0))), __float_as_uint(fabsf(a1)));   // as integers: a NaN wins
        vtb = max(max(vtb, __float_as_uint(b0)), __float_as_uint(b1));
        gt = fmaxf(fmaxf(gt, fabsf(g[h][k])), fabsf(g[h][k + 1]));
        // the update itself with the one-instruction root and reciprocal (2 kU each): its error
        // is far below that of the 8-bit states it is made from
        float d0, d1;
        fma2(F2(sqrt_ftz(b0), sqrt_ftz(b1)), F2(c.inv_root), F2(a.eps)).split(d0, d1);
        fma2(F2(-c.step), mm * F2(rcp_ftz(d0), rcp_ftz(d1)), F2(p[h][k], p[h][k + 1]) * F2(c.decay)).split(p[h][k], p[h][k + 1]);
      }
      store4<P>(t.p, i[h], nv[h], vec, p[h]);
      if (sizeof(P) == 4 && t.shadow) store4<__nv_bfloat16>(t.shadow, i[h], nv[h], vec, p[h]);
    }
    const float mt = __uint_as_float(__reduce_max_sync(0xffffffffu, mtb));
    const float vt = __uint_as_float(__reduce_max_sync(0xffffffffu, vtb));
    // no |old term| + |new term| of the block is above et
    gt = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(gt)));
    const float et = 1.0001f * fmaf(gt, o1, 16129.f * cm);
    // fp32 carries the block where its largest values are well inside the range and the means
    // do not cancel throughout; an all-zero block is exact
    const bool mok = (mt > 0x1p-90f && mt < 0x1p100f && et <= 32.f * mt) || et == 0.f;
    const bool vok = (vt > 0x1p-70f && vt < 0x1p100f && (vs == 0.f || vs > 0x1p-60f)) ||
                     (vt == 0.f && gt == 0.f && !__any_sync(0xffffffffu, (vq[0] | vq[1]) != 0));
    const float im = mt > 0.f ? 16129.f * rcp_ftz(mt) : 0.f, iv = vt > 0.f ? 4228250625.f * rcp_ftz(vt) : 0.f;
    const float ir = sqrt_ftz(iv);
    // error of y = |m| im: at most 4 kU et im from m, and relative 4 kU et / mt from the top, 3 kU
    // from the quotient, 1 from the product and 2 of second order
    const float e0 = 4.f * kU * im * et, ey = kU * (4.f * et * rcp_ftz(mt) + 6.f);
    // y = (127 sqrt(|m| / top))^2 of a pair lies next to the borders b^2, b = floor(sqrt(y)) + 1/2,
    // which split the codes b - 1/2 and b + 1/2; returns b, y - b^2 and the error of that
    auto mean_border = [&](F2 m, F2& b, F2& d, F2& tol) {
      float a0, a1, y0, y1;
      m.split(a0, a1);
      const F2 y = F2(fabsf(a0), fabsf(a1)) * F2(im);
      y.split(y0, y1);
      b = add_down(F2(sqrt_ftz(y0), sqrt_ftz(y1)), F2(8388608.f)) + F2(-8388607.5f);
      float c0, c1;
      b.split(c0, c1);
      d = fma2(F2(-c0, -c1), b, y);                                       // b^2 is exact
      tol = fma2(F2(ey), y, F2(e0));
    };
    // likewise b^4 and z = (255 sqrt(sqrt(v) / top))^4: relative 6 kU for v, 6 for the top, 4 for
    // the quotient and its product, 2 for the border
    auto root_border = [&](F2 v, F2& b, F2& d, F2& tol) {
      float a0, a1, x0, x1;
      v.split(a0, a1);
      (F2(sqrt_ftz(a0), sqrt_ftz(a1)) * F2(ir)).split(x0, x1);
      b = add_down(F2(sqrt_ftz(x0), sqrt_ftz(x1)), F2(8388608.f)) + F2(-8388607.5f);
      const F2 r2 = b * b;
      float s0, s1;
      r2.split(s0, s1);
      d = fma2(F2(-s0, -s1), r2, v * F2(iv));
      tol = (r2 * F2(20.f * kU)) * r2;
    };
    bool near = false;             // an element of this lane lies next to a border
    uint32_t um[2], uv[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t qm[4], qv[4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        F2 b, d, tol;
        float b0, b1, d0, d1, t0, t1, s0, s1;
        mean_border(m2[h][j], b, d, tol);
        d.split(d0, d1);
        tol.split(t0, t1);
        m2[h][j].split(s0, s1);
        near |= fabsf(d0) <= t0;
        near |= fabsf(d1) <= t1;
        (b + F2(copysignf(0.5f, d0), copysignf(0.5f, d1))).split(b0, b1);
        // the low byte of 1.5 2^23 + q is q's two's complement
        (F2(copysignf(b0, s0), copysignf(b1, s1)) + F2(12582912.f)).split(b0, b1);
        qm[2 * j] = __float_as_uint(b0);
        qm[2 * j + 1] = __float_as_uint(b1);
        root_border(v2[h][j], b, d, tol);
        d.split(d0, d1);
        tol.split(t0, t1);
        near |= fabsf(d0) <= t0;
        near |= fabsf(d1) <= t1;
        (b + F2(copysignf(0.5f, d0), copysignf(0.5f, d1)) + F2(8388608.f)).split(b0, b1);
        qv[2 * j] = __float_as_uint(b0);
        qv[2 * j + 1] = __float_as_uint(b1);
      }
      um[h] = pack4(qm);
      uv[h] = pack4(qv);
      if (((uv[h] - 0x01010101u) & ~uv[h] & 0x80808080u) != 0) {          // a code 0: a positive v keeps 1
        float raw[4];                                    // the gradient before a scale that may underflow
        load4<G>(t.g, i[h], nv[h], vec, raw);
        const bool live = !a.grad_scale || *a.grad_scale != 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if ((uv[h] >> (8 * k) & 0xFFu) == 0 && ((raw[k] != 0.f && live) || (vq[h] >> (8 * k) & 0xFFu) != 0)) uv[h] |= 1u << (8 * k);
      }
    }
    float msn = 0.f, vsn = 0.f;
    if (!(mok && vok)) {
      exact_block<G>(t, base, lane, a.b1, a.omb1, a.b2, a.omb2, a.grad_scale, um, uv, msn, vsn);
    } else {
      // The scales come from the largest values in fp64. Lanes whose largest could be it in spite
      // of the roundings (nearly always one): their eight elements are formed again, side by side
      // on eight lanes, lanes 0-7 for m and 8-15 for v.
      uint32_t cand_m = __ballot_sync(0xffffffffu, mt > 0.f && __uint_as_float(mtb) >= mt - 8.f * kU * et);
      uint32_t cand_v = __ballot_sync(0xffffffffu, vt > 0.f && __uint_as_float(vtb) >= vt * (1.f - 16.f * kU));
      const double gs64 = a.grad_scale ? static_cast<double>(*a.grad_scale) : 1.0;
      auto grad_at = [&](int64_t at) {
        return sizeof(G) == 4 ? reinterpret_cast<const float*>(t.g)[at]
                              : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(t.g)[at]);
      };
      auto m64_at = [&](int64_t at) {
        return mean64(reinterpret_cast<const int8_t*>(t.m)[at], ms, grad_at(at), gs64, a.b1, a.omb1);
      };
      auto v64_at = [&](int64_t at) {
        return root64(reinterpret_cast<const uint8_t*>(t.v)[at], vs, grad_at(at), gs64, a.b2, a.omb2);
      };
      double top64 = 0.0;
      if (__popc(cand_m) + __popc(cand_v) <= 8) {
        while ((cand_m | cand_v) != 0) {
          const int src = __ffs(static_cast<int>((lane & 8) ? cand_v : cand_m)) - 1;
          const int64_t at = base + 128 * ((lane >> 2) & 1) + 4 * src + (lane & 3);
          if (src >= 0 && lane < 16 && (FULL || at < t.n)) top64 = fmax(top64, (lane & 8) ? v64_at(at) : fabs(m64_at(at)));
          cand_m &= cand_m - 1;
          cand_v &= cand_v - 1;
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top64 = fmax(top64, __shfl_xor_sync(0xffffffffu, top64, o));
      } else {                                           // many equal values: every element again
        double m64 = 0.0, v64 = 0.0;
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const int64_t at = base + 128 * (e >> 2) + 4 * lane + (e & 3);
          if (FULL || at < t.n) {
            m64 = fmax(m64, fabs(m64_at(at)));
            v64 = fmax(v64, v64_at(at));
          }
        }
        m64 = warp_top(m64);
        v64 = warp_top(v64);
        top64 = (lane & 8) ? v64 : m64;
      }
      msn = static_cast<float>(top64 * (1.0 / 16129.0));                  // lanes 0-7
      // lanes 8-15: two Newton steps take the fp32 root (2^-23) to fp64's last bits
      const float r0 = sqrt_ftz(static_cast<float>(top64));
      const double half = static_cast<double>(0.5f * rcp_ftz(r0));
      double r1 = static_cast<double>(r0);
      if (r0 > 0.f) {
        r1 = fma(fma(-r1, r1, top64), half, r1);
        r1 = fma(fma(-r1, r1, top64), half, r1);
      }
      vsn = __shfl_sync(0xffffffffu, static_cast<float>(r1 * (1.0 / 65025.0)), 8);
      if (__any_sync(0xffffffffu, near)) {
        // codes of the elements next to a border (a block in thirty has one) from fp64
        const double mt64 = __shfl_sync(0xffffffffu, top64, 0), vt64 = __shfl_sync(0xffffffffu, top64, 8);
        uint32_t which = 0;                              // bits 0-7 for m, 8-15 for v
        if (near) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            F2 b, d, tol;
            float d0, d1, t0, t1;
            mean_border(m2[e >> 1][e & 1], b, d, tol);
            d.split(d0, d1);
            tol.split(t0, t1);
            which |= (fabsf(d0) <= t0 ? 1u << (2 * e) : 0u) | (fabsf(d1) <= t1 ? 2u << (2 * e) : 0u);
            root_border(v2[e >> 1][e & 1], b, d, tol);
            d.split(d0, d1);
            tol.split(t0, t1);
            which |= (fabsf(d0) <= t0 ? 256u << (2 * e) : 0u) | (fabsf(d1) <= t1 ? 512u << (2 * e) : 0u);
          }
        }
        while (which != 0) {
          const int e = __ffs(static_cast<int>(which)) - 1, k = e & 3;
          which &= which - 1;
          const int64_t at = base + 128 * ((e >> 2) & 1) + 4 * lane + k;
          uint32_t q, clear = ~(0xFFu << (8 * k));
          if (e < 8) {
            const double m64 = m64_at(at);
            const int qi = mean_code(fabs(m64), mt64);
            q = (static_cast<uint32_t>(m64 < 0.0 ? -qi : qi) & 0xFFu) << (8 * k);
            if (e < 4) um[0] = (um[0] & clear) | q; else um[1] = (um[1] & clear) | q;
          } else {
            q = static_cast<uint32_t>(root_code(v64_at(at), __dsqrt_rn(vt64))) << (8 * k);
            if (e < 12) uv[0] = (uv[0] & clear) | q; else uv[1] = (uv[1] & clear) | q;
          }
        }
        __syncwarp();
      }
    }
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
}

// 8-bit states: 32 warps an SM, 64 registers a thread. (In CTAs of 256 threads, before packed
// arithmetic: 628 us for a 7B set so, 739 with 24 warps, 840 with 40.)
template <int CAP, typename P, typename G, int BITS>
__global__ void __launch_bounds__(kThreadsAW, BITS == 8 ? 16 : 1) k_adamw(const __grid_constant__ Args<CAP> a) {
  const int ti = tensor_of(a, static_cast<int>(blockIdx.x));
  const Tensor& t = a.t[ti];
  const int lane = threadIdx.x & 31;
  const bool vec = a.vec[ti] != 0;
  const int64_t base = static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.tile0[ti]) * kTile + (threadIdx.x >> 5) * kBlock;
  if (base >= t.n) return;                         // the whole warp: no element of this block exists
  if (vec && base + kBlock <= t.n) step_block<CAP, P, G, BITS, true>(a, t, base, lane, true);
  else step_block<CAP, P, G, BITS, false>(a, t, base, lane, vec);
}

// The fp32 values that 8-bit codes stand for.
template <int CAP>
__global__ void __launch_bounds__(kThreadsAW) k_adamw_values(const __grid_constant__ Args<CAP> a) {
  const int ti = tensor_of(a, static_cast<int>(blockIdx.x));
  const Tensor& t = a.t[ti];
  const int lane = threadIdx.x & 31;
  const bool vec = a.vec[ti] != 0;
  int64_t base = (static_cast<int64_t>(static_cast<int>(blockIdx.x) - a.tile0[ti]) * a.tiles) * kTile +
                 (threadIdx.x >> 5) * kBlock;
  for (int j = 0; j < a.tiles && base < t.n; ++j, base += kTile) {
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
}

}  // namespace aw
}  // namespace dsmz
