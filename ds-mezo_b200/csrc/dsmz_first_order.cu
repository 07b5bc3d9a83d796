// C ABI of the first-order operators declared in dsmezo.h: products grouped by adapter copy,
// the scoring loss with its gradient, and AdamW over many tensors.
#include <atomic>
#include <cmath>
#include <exception>
#include <vector>

#include "dsmezo.h"
#include "dsmz_adamw.cuh"
#include "dsmz_grouped.cuh"
#include "dsmz_host.h"
#include "dsmz_score_grad.cuh"

using namespace dsmz;

namespace {

constexpr int64_t kMaxElems = int64_t{1} << 40;

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(const char* what, F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    try {
      return fail(DSMZ_ERR_INVALID, std::string(what) + ": " + e.what());
    } catch (...) {
      return DSMZ_ERR_INVALID;
    }
  } catch (...) {
    return DSMZ_ERR_INVALID;
  }
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// ------------------------------------------------------------------ AdamW
// Tensors per launch: the argument block (by value) of the small form is 0.6 KB, so that a
// call on a few tensors does not pay for copying the large one (18 KB).
constexpr int kSmall = 8, kLarge = 256;
// Reading states back takes four tiles a CTA where that still fills the machine four times over
// (289 -> 267 us for a 7B set: a tile is short against finding its tensor in the arguments).
// The step does not: a second tile's loads would wait for the first (8-bit 634 -> 784 us; with
// them issued ahead and three CTAs an SM for the registers, 688).
constexpr int64_t kManyTiles = 148 * 16 * 4;

template <int CAP>
void launch_adamw(const aw::Args<CAP>& a, int grid, int pdt, int gdt, int bits, cudaStream_t s) {
  using bf = __nv_bfloat16;
  const int t = aw::kThreadsAW;
  if (bits == 32) {
    if (pdt == DSMZ_F32 && gdt == DSMZ_F32) aw::k_adamw<CAP, float, float, 32><<<grid, t, 0, s>>>(a);
    else if (pdt == DSMZ_F32) aw::k_adamw<CAP, float, bf, 32><<<grid, t, 0, s>>>(a);
    else if (gdt == DSMZ_F32) aw::k_adamw<CAP, bf, float, 32><<<grid, t, 0, s>>>(a);
    else aw::k_adamw<CAP, bf, bf, 32><<<grid, t, 0, s>>>(a);
  } else {
    if (pdt == DSMZ_F32 && gdt == DSMZ_F32) aw::k_adamw<CAP, float, float, 8><<<grid, t, 0, s>>>(a);
    else if (pdt == DSMZ_F32) aw::k_adamw<CAP, float, bf, 8><<<grid, t, 0, s>>>(a);
    else if (gdt == DSMZ_F32) aw::k_adamw<CAP, bf, float, 8><<<grid, t, 0, s>>>(a);
    else aw::k_adamw<CAP, bf, bf, 8><<<grid, t, 0, s>>>(a);
  }
}

// Launches over tensors[0..n): as many per launch as CAP and the grid limit allow.
template <int CAP, typename Fill, typename Launch>
int chunked(const dsmz_adamw_tensor* tensors, int32_t n, int tiles_max, const char* what, Fill fill, Launch launch) {
  auto box = std::vector<aw::Args<CAP>>(1);
  aw::Args<CAP>& a = box[0];
  int64_t all = 0;
  for (int32_t k = 0; k < n; ++k) all += (tensors[k].n + aw::kTile - 1) / aw::kTile;
  a.tiles = all >= tiles_max * kManyTiles ? tiles_max : 1;
  const int64_t per = static_cast<int64_t>(a.tiles) * aw::kTile;
  int32_t i = 0;
  while (i < n) {
    a.n = 0;
    int64_t tiles = 0;
    for (; i < n && a.n < CAP; ++i) {
      if (tensors[i].n == 0) continue;
      const int64_t nt = (tensors[i].n + per - 1) / per;
      if (tiles + nt > 0x7fffffff) {
        if (a.n > 0) break;
        return fail(DSMZ_ERR_UNSUPPORTED, std::string(what) + ": a tensor with too many elements");
      }
      fill(a, a.n, tensors[i]);
      a.tile0[a.n] = static_cast<int32_t>(tiles);
      tiles += nt;
      a.tile0[++a.n] = static_cast<int32_t>(tiles);
    }
    if (tiles > 0) {
      launch(a, static_cast<int>(tiles));
      DSMZ_LAUNCHED(what);
    }
  }
  return DSMZ_OK;
}

int check_tensors(const char* what, const dsmz_adamw_tensor* t, int32_t n, int bits, bool values, int pdt, int gdt) {
  if (n < 0 || (n > 0 && !t)) return fail(DSMZ_ERR_INVALID, std::string(what) + ": null tensor list");
  const size_t ps = pdt == DSMZ_F32 ? 4 : 2, gs = gdt == DSMZ_F32 ? 4 : 2;
  for (int32_t i = 0; i < n; ++i) {
    const char* bad = nullptr;
    const dsmz_adamw_tensor& x = t[i];
    if (x.n < 0 || x.n > kMaxElems) bad = " has a bad element count";
    else if (x.n == 0) continue;
    else if (!x.param || !x.m || !x.v || (values ? !x.shadow : !x.grad)) bad = " has a null pointer";
    else if (bits == 8 && (!x.m_scale || !x.v_scale)) bad = ": 8-bit states need scales";
    else if (!aligned(x.param, ps) || (!values && !aligned(x.grad, gs)) || (x.shadow && !aligned(x.shadow, values ? 4 : 2)) ||
             (bits == 32 && (!aligned(x.m, 4) || !aligned(x.v, 4))) ||
             (bits == 8 && (!aligned(x.m_scale, 4) || !aligned(x.v_scale, 4))))
      bad = " is not aligned to its element type";
    else if (x.shadow && !values && pdt != DSMZ_F32) bad = ": a shadow belongs to fp32 parameters";
    if (bad) return fail(DSMZ_ERR_INVALID, std::string(what) + ": tensor " + std::to_string(i) + bad);
  }
  return DSMZ_OK;
}

template <int CAP>
int adamw_values(const dsmz_adamw_tensor* tensors, int32_t n, cudaStream_t s) {
  return chunked<CAP>(
      tensors, n, 4, "dsmz_adamw_state_values",
      [](aw::Args<CAP>& a, int k, const dsmz_adamw_tensor& t) {
        a.t[k] = aw::Tensor{t.param, nullptr, t.m, t.v, t.m_scale, t.v_scale, t.shadow, t.n};
        a.vec[k] = aligned(t.param, 16) && aligned(t.shadow, 16) && aligned(t.m, 4) && aligned(t.v, 4);
      },
      [&](const aw::Args<CAP>& a, int grid) { aw::k_adamw_values<CAP><<<grid, aw::kThreadsAW, 0, s>>>(a); });
}

template <int CAP>
int adamw_run(const dsmz_adamw_desc& d, const dsmz_adamw_tensor* tensors, int32_t n, const aw::Coef& c,
              const aw::Coef* dc, cudaStream_t s) {
  const size_t pa = d.param_dtype == DSMZ_F32 ? 16 : 8, ga = d.grad_dtype == DSMZ_F32 ? 16 : 8;
  const size_t sa = d.state_bits == 32 ? 16 : 4;
  return chunked<CAP>(
      tensors, n, 1, "dsmz_adamw_step",
      [&](aw::Args<CAP>& a, int k, const dsmz_adamw_tensor& t) {
        a.b1 = d.beta1; a.omb1 = 1.0 - d.beta1;
        a.b2 = d.beta2; a.omb2 = 1.0 - d.beta2;
        a.fb1 = static_cast<float>(a.b1); a.fo1 = static_cast<float>(a.omb1);
        a.fb2 = static_cast<float>(a.b2); a.fo2 = static_cast<float>(a.omb2);
        a.eps = static_cast<float>(d.eps);
        a.c = c;
        a.dc = dc;
        a.grad_scale = d.grad_scale;
        a.t[k] = aw::Tensor{t.param, t.grad, t.m, t.v, t.m_scale, t.v_scale, t.shadow, t.n};
        a.vec[k] = aligned(t.param, pa) && aligned(t.grad, ga) && aligned(t.m, sa) && aligned(t.v, sa) &&
                   aligned(t.shadow, 8);
      },
      [&](const aw::Args<CAP>& a, int grid) { launch_adamw<CAP>(a, grid, d.param_dtype, d.grad_dtype, d.state_bits, s); });
}

// Error word of the bounded waits, one per device, and their limit.
__device__ int g_wait_err;
std::atomic<int64_t> g_wait_ns{static_cast<int64_t>(kTimeoutNs)};

int wait_err(int** p) {
  void* q = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&q, g_wait_err);
  *p = static_cast<int*>(q);
  return e == cudaSuccess ? 0 : cuda_fail("error word", e);
}

// ------------------------------------------------------------------ products grouped by adapter copy

// Tensor map of rank 2 to 4 (inner dimension contiguous, byte strides of the others, boxes of up
// to three dimensions), 128-byte swizzle, zero fill outside; bf16, or fp32.
bool encode_map(CUtensorMap* m, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                uint32_t box0, uint32_t box1, bool f32 = false, uint32_t box2 = 1) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[4] = {1, 1, 1, 1}, st[3] = {0, 0, 0};
  for (int i = 0; i < rank; ++i) d[i] = dims[i];
  for (int i = 0; i + 1 < rank; ++i) st[i] = strides[i];
  cuuint32_t box[4] = {box0, box1, box2, 1}, es[4] = {1, 1, 1, 1};
  return fn(m, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, static_cast<cuuint32_t>(rank),
            const_cast<void*>(base), d, st, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// `rows` rows of `width` bf16 (byte pitch), to be read in boxes of 64 rows x `cols` columns with the
// column as the MMA's major dimension: slabs of 64 columns (64, row, slab) where the width is a
// whole number of them, so that a box is one copy; else boxes of 64 columns.
bool encode_width(CUtensorMap* m, int32_t* slabs, const void* base, int64_t width, int64_t rows, int64_t pitch, int cols) {
  *slabs = width % 64 == 0;
  const uint64_t d[3] = {*slabs ? 64u : static_cast<uint64_t>(width), static_cast<uint64_t>(rows), static_cast<uint64_t>(width / 64)};
  const uint64_t st[2] = {static_cast<uint64_t>(pitch) * 2, 128};
  return *slabs ? encode_map(m, base, 3, d, st, 64, 64, false, static_cast<uint32_t>((cols + 63) / 64))
                : encode_map(m, base, 2, d, st, 64, 64);
}

int sm_count(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
  return e == cudaSuccess ? 0 : cuda_fail("device query", e);
}

// Shared memory of a launch; sets a.sbuf and a.stages.
template <int BNT, int MODE, bool PAIR, int EW>
size_t grouped_smem(gr::Args& a, int64_t nk) {
  constexpr int SB = gr::kABytes + (PAIR ? BNT / 2 : BNT) * gr::kBK * 2;
  constexpr int kSmem = 227 * 1024;
  // two staging pieces a warp let a store run while the next piece is staged; the widest tile
  // gives a stage of the ring for them, which pays where a tile has only a few k-steps
  a.sbuf = EW == 8 && (BNT < 256 || PAIR || nk <= 4) ? 2 : 1;
  const int scratch = a.split > 1 ? gr::split_bytes(a.split, BNT) : EW * gr::kStageBytes * a.sbuf;
  const int fixed = 1024 + scratch + (((a.G + 3) * 8 + 15) & ~15) + 64 + 16 * 8;
  a.stages = (kSmem - fixed) / SB;
  if (a.stages > 8) a.stages = 8;
  return static_cast<size_t>(fixed) + static_cast<size_t>(a.stages) * SB;
}

template <int BNT, int MODE, bool PAIR, bool SUM, int EW = 8>
int launch_grouped(gr::Args a, const CUtensorMap& A, const CUtensorMap& B, const CUtensorMap& C, int64_t tiles, int64_t nk,
                   int sms, const char* what, cudaStream_t s) {
  const size_t smem = grouped_smem<BNT, MODE, PAIR, EW>(a, nk);
  a.wait_ns = static_cast<uint64_t>(g_wait_ns.load(std::memory_order_relaxed));
  auto* kernel = gr::k_grouped<BNT, MODE, PAIR, SUM, EW>;
  int* err = nullptr;
  int rc = wait_err(&err);
  if (rc) return rc;
  static thread_local int set_dev = -1;                  // the device whose shared memory limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev != set_dev) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e == cudaSuccess) set_dev = dev;
  }
  if (e != cudaSuccess) return cuda_fail(what, e);
  cudaLaunchConfig_t cfg{};
  const int cluster = PAIR ? 2 : a.split;
  const int64_t wave = sms / 2;                          // pairs: one a TPC
  cfg.gridDim = dim3(static_cast<unsigned>(PAIR ? 2 * (tiles < wave ? tiles : wave)
                                                : (a.split > 1 ? tiles * a.split : (tiles < sms ? tiles : sms))));
  cfg.blockDim = dim3(32 * (gr::kFirstEpi + EW));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, kernel, A, B, C, a, err);
  return e == cudaSuccess ? DSMZ_OK : cuda_fail(what, e);
}

template <int MODE, bool SUM>
int launch_grouped_bn(int bnt, const gr::Args& a, const CUtensorMap& A, const CUtensorMap& B, const CUtensorMap& C,
                      int64_t tiles, int64_t nk, int sms, const char* what, cudaStream_t s) {
  if (bnt == 64) return launch_grouped<64, MODE, false, SUM>(a, A, B, C, tiles, nk, sms, what, s);
  if (bnt == 128) return launch_grouped<128, MODE, false, SUM>(a, A, B, C, tiles, nk, sms, what, s);
  return launch_grouped<256, MODE, false, SUM>(a, A, B, C, tiles, nk, sms, what, s);
}

// Accumulator width for n output columns and `rows` row tiles: 256 columns where that still
// gives every SM a tile.
int columns_for(int64_t n, int64_t rows, int sms) {
  if (n <= 64) return 64;
  if (n <= 128) return 128;
  return rows * ((n + 255) / 256) >= sms ? 256 : 128;
}
// Clusters of s CTAs (one CTA an SM) that the current device runs at once. A cluster lies inside
// one GPC, whose SMs it need not divide: 74, 45, 33, 26, 22, 15 and 15 clusters of 2 to 8 on a
// chip with 148 SMs.
int active_clusters(int s) {
  static thread_local int cached[9] = {0}, cached_dev = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev != cached_dev) {
    for (int c = 2; c <= 8; ++c) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(static_cast<unsigned>(c * 256));
      cfg.blockDim = dim3(32 * (gr::kFirstEpi + 8));
      cfg.dynamicSmemBytes = 200 * 1024;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = static_cast<unsigned>(c);
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      auto* kernel = gr::k_grouped<128, 0, false, false, 8>;
      int n = 0;
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess ||
          cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;                                           // not known: no split of this size
      }
      cached[c] = n;
    }
    cached_dev = dev;
  }
  return cached[s];
}

// CTAs that share a tile's contraction: as many as one wave of clusters allows, while each still
// has two k-steps. A second wave would double the time (the 70B rank gradient, 36 tiles in
// clusters of 4: 93 us).
int split_for(int bnt, int64_t tiles, int64_t nk) {
  if (bnt > 128) return 1;
  for (int s = 8; s > 1; --s)
    if (tiles <= active_clusters(s) && nk / s >= 2) return s;
  return 1;
}

// Whether `rows` rows of `na` bytes at a and of `nb` bytes at b share a byte; rows of one pitch may lie
// side by side in a wider buffer. With two pitches: whether their ranges meet.
bool rows_meet(const void* a, int64_t na, int64_t pitch_a, const void* b, int64_t nb, int64_t pitch_b, int64_t rows) {
  const int64_t x = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a)), y = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b));
  const int64_t all_a = (rows - 1) * pitch_a + na, all_b = (rows - 1) * pitch_b + nb;
  if (x + all_a <= y || y + all_b <= x) return false;
  if (rows < 2 || pitch_a != pitch_b) return true;
  const int64_t d = ((y - x) % pitch_a + pitch_a) % pitch_a;   // where b's rows begin between two of a's
  return d < na || d + nb > pitch_a;
}
bool overlaps(const void* a, int64_t na, const void* b, int64_t nb) { return rows_meet(a, na, 0, b, nb, 0, 1); }

// ------------------------------------------------------------------ scoring loss with its gradient
template <typename T>
int loss_grad(const void* logits, int64_t V, int64_t ld, const int32_t* targets, int64_t ntok, const sg::Seqs& q,
              double grad_scale, float* loss, void* grad, int64_t ld_grad, double* term, cudaStream_t s) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return cuda_fail("dsmz_contrastive_loss_grad: device query", e);
  // CTAs a row: slices of at most kSliceBytes, and more where a few rows would leave SMs idle
  // while a slice is still worth a CTA
  const int64_t row_bytes = V * static_cast<int64_t>(sizeof(T));
  int C = 1;
  while (C < 8 && (row_bytes / C > sg::kSliceBytes || (ntok * C < 2 * sms && row_bytes / C > 8192))) C *= 2;
  const int64_t vecs = (row_bytes / C + 15) / 16;
  const int threads = vecs >= 256 ? 256 : 128;
  if (ntok * C > 0x7fffffff) return fail(DSMZ_ERR_UNSUPPORTED, "dsmz_contrastive_loss_grad: too many tokens");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ntok * C));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = static_cast<unsigned>(C);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, sg::k_loss_grad<T>, static_cast<const T*>(logits), ld, V, targets, q, grad_scale,
                         static_cast<T*>(grad), ld_grad, term);
  if (e != cudaSuccess) return cuda_fail("dsmz_contrastive_loss_grad: rows", e);
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(256);
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  e = cudaLaunchKernelEx(&cfg, sg::k_loss_sum, static_cast<const double*>(term), ntok, loss);
  return e == cudaSuccess ? DSMZ_OK : cuda_fail("dsmz_contrastive_loss_grad: sum", e);
}

}  // namespace

extern "C" {

int dsmz_grouped_matmul(const void* x, int64_t M, int64_t K, int64_t ld_x, const void* w, int32_t G, int64_t N,
                        int64_t w_group_stride, int64_t w_ld, int32_t w_n_contiguous, const int32_t* row_offsets,
                        int32_t out_dtype, void* out, int64_t ld_out, float alpha, uint32_t flags,
                        dsmz_stream_t stream) {
  return guarded("dsmz_grouped_matmul", [&]() -> int {
    const std::string me = "dsmz_grouped_matmul: ";
    if (M < 0 || K < 1 || N < 1 || G < 1) return fail(DSMZ_ERR_INVALID, me + "need M >= 0, K >= 1, N >= 1 and G >= 1");
    if (G > DSMZ_MAX_GROUPS || M > DSMZ_MAX_GROUPED_DIM || K > DSMZ_MAX_GROUPED_DIM || N > DSMZ_MAX_GROUPED_DIM)
      return fail(DSMZ_ERR_UNSUPPORTED, me + "at most DSMZ_MAX_GROUPS groups and DSMZ_MAX_GROUPED_DIM rows or columns");
    if (out_dtype != DSMZ_F32 && out_dtype != DSMZ_BF16) return fail(DSMZ_ERR_INVALID, me + "out must be DSMZ_F32 or DSMZ_BF16");
    if (flags & ~(DSMZ_GROUPED_ACCUMULATE | DSMZ_GROUPED_ZERO_REST)) return fail(DSMZ_ERR_INVALID, me + "unknown flag");
    if (M == 0) return DSMZ_OK;
    if (!x || !w || !row_offsets || !out) return fail(DSMZ_ERR_INVALID, me + "null pointer");
    const int64_t wi = w_n_contiguous ? N : K, wo = w_n_contiguous ? K : N;      // inner and outer width of W_g
    const int es = out_dtype == DSMZ_F32 ? 4 : 2;
    if (ld_x < K || w_ld < wi || ld_out < N || (G > 1 && w_group_stride < 1) || ld_x > kMaxElems || w_ld > kMaxElems ||
        ld_out > kMaxElems || w_group_stride > kMaxElems)
      return fail(DSMZ_ERR_INVALID, me + "a pitch is smaller than its row, or a stride is out of range");
    if (!aligned(x, 16) || !aligned(w, 16) || ld_x % 8 || w_ld % 8 || (G > 1 && w_group_stride % 8))
      return fail(DSMZ_ERR_INVALID, me + "x and w need 16-byte aligned bases and strides that are multiples of 8 elements");
    if (!aligned(out, es) || !aligned(row_offsets, 4)) return fail(DSMZ_ERR_INVALID, me + "a pointer is not aligned to its type");
    if (!std::isfinite(alpha)) return fail(DSMZ_ERR_INVALID, me + "alpha must be finite");
    const int64_t nout = ((M - 1) * ld_out + N) * es;
    if (rows_meet(out, N * es, ld_out * es, x, K * 2, ld_x * 2, M) || overlaps(out, nout, w, ((G - 1) * w_group_stride + (wo - 1) * w_ld + wi) * 2))
      return fail(DSMZ_ERR_INVALID, me + "out overlaps an operand");
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    gr::Args a{};
    a.offsets = row_offsets;
    a.G = G;
    a.M = M;
    a.ndim = static_cast<int32_t>(N);
    a.kdim = static_cast<int32_t>(K);
    a.b_mn = w_n_contiguous ? 1 : 0;
    a.n_inner = K <= 256 ? 1 : 0;
    a.out = out;
    a.ld = ld_out;
    a.out_f32 = out_dtype == DSMZ_F32;
    a.accumulate = (flags & DSMZ_GROUPED_ACCUMULATE) ? 1 : 0;
    a.zero_rest = (flags & DSMZ_GROUPED_ZERO_REST) && !a.accumulate;
    a.vec = aligned(out, 16) && (ld_out * es) % 16 == 0;
    a.alpha = alpha;
    const int64_t rows = (M + gr::kBM - 1) / gr::kBM + (G < M ? G : M) - 1;      // most row tiles the groups can have
    const int bnt = columns_for(N, rows, sms);
    a.bn = static_cast<int32_t>(N >= bnt ? bnt : (N + 15) / 16 * 16);
    a.ntn = static_cast<int32_t>((N + a.bn - 1) / a.bn);
    const int64_t nk = (K + gr::kBK - 1) / gr::kBK;
    a.split = split_for(bnt, rows * a.ntn, nk);
    const bool sum = a.out_f32 || (nk + a.split - 1) / a.split > gr::kLong;
    a.chunk = sum ? gr::kChunk : 0x3fffffff;
    // Pairs of CTAs where the products, not the output, take a tile's time and the groups are long
    // enough for 256-row tiles. 8192 x 3584 x 18944 in 8 ragged groups (9% of the tiles' rows are
    // empty, 5% with 128-row tiles): 826 us with pairs and 856 without in a short run, 1014 and
    // 1078 under the power cap.
    const bool pair = bnt == 256 && N >= 256 && K >= 512 && M / G >= 512 && rows / 2 * a.ntn >= sms / 2;
    // short groups: boxes of 32 rows, so that a tile does not fetch 128
    a.arows = M / G >= 96 ? gr::kBM : 32;
    const int64_t tiles = (rows + 2) * a.ntn;                                    // and the rows outside the groups
    const uint32_t bcols = static_cast<uint32_t>(pair ? a.bn / 2 : a.bn);        // columns of a CTA's box of W
    if (tiles > (1 << 27)) return fail(DSMZ_ERR_UNSUPPORTED, me + "too many tiles");
    CUtensorMap A, B, C{};
    const uint64_t da[2] = {static_cast<uint64_t>(K), static_cast<uint64_t>(M)}, sa[1] = {static_cast<uint64_t>(ld_x) * 2};
    const uint64_t pitch = static_cast<uint64_t>(w_ld) * 2;
    const uint64_t group = static_cast<uint64_t>(G > 1 ? w_group_stride : (w_ld * wo + 7) / 8 * 8) * 2;
    const uint64_t db[3] = {static_cast<uint64_t>(wi), static_cast<uint64_t>(wo), static_cast<uint64_t>(G)}, sb[2] = {pitch, group};
    const uint64_t ds[4] = {64, static_cast<uint64_t>(wo), static_cast<uint64_t>(wi / 64), static_cast<uint64_t>(G)};
    const uint64_t ss[3] = {pitch, 128, group};
    a.b_slabs = w_n_contiguous && N % 64 == 0;
    if (!encode_map(&A, x, 2, da, sa, gr::kBK, static_cast<uint32_t>(a.arows)) ||
        !(a.b_slabs ? encode_map(&B, w, 4, ds, ss, 64, 64, false, (bcols + 63) / 64)
                    : encode_map(&B, w, 3, db, sb, 64, w_n_contiguous ? 64 : bcols)))
      return fail(DSMZ_ERR_CUDA, me + "the driver refused a tensor map");
    if (a.vec && !a.accumulate && a.split == 1 && (a.out_f32 || !sum)) {
      const uint64_t dc[3] = {static_cast<uint64_t>(N), static_cast<uint64_t>(M), 1};
      const uint64_t sc[2] = {static_cast<uint64_t>(ld_out) * es, static_cast<uint64_t>(ld_out) * es * M};
      a.tma_out = encode_map(&C, out, 3, dc, sc, 128 / es, 32, a.out_f32 != 0);
    }
    const char* what = "dsmz_grouped_matmul";
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (sum)
      return pair ? launch_grouped<256, 0, true, true>(a, A, B, C, tiles, nk, sms, what, s)
                  : launch_grouped_bn<0, true>(bnt, a, A, B, C, tiles, nk, sms, what, s);
    // Few k-steps and short groups: a tile's epilogue sets the pace, and 16 warps shorten it. K = 64, N =
    // 18944, 32 groups of 64, 127, 160 rows: 28.0, 45.5, 52.8 us with 16 and 31.8, 46.7, 56.0 with 8;
    // with 192, 256 and 512 rows, where the stores' bandwidth does, 68, 83, 142 and 56, 81, 139. (Rows of
    // no group count in M / G: the host does not know the offsets.)
    if (bnt == 256 && nk <= 4 && M / G <= 160) return launch_grouped<256, 0, false, false, 16>(a, A, B, C, tiles, nk, sms, what, s);
    return pair ? launch_grouped<256, 0, true, false>(a, A, B, C, tiles, nk, sms, what, s)
                : launch_grouped_bn<0, false>(bnt, a, A, B, C, tiles, nk, sms, what, s);
  });
}

int dsmz_grouped_weight_grad(const void* x, int64_t M, int64_t K, int64_t ld_x, const void* dy, int64_t N, int64_t ld_dy,
                             int32_t G, const int32_t* row_offsets, float* out, float alpha, uint32_t flags,
                             dsmz_stream_t stream) {
  return guarded("dsmz_grouped_weight_grad", [&]() -> int {
    const std::string me = "dsmz_grouped_weight_grad: ";
    if (M < 0 || K < 1 || N < 1 || G < 1) return fail(DSMZ_ERR_INVALID, me + "need M >= 0, K >= 1, N >= 1 and G >= 1");
    if (G > DSMZ_MAX_GROUPS || M > DSMZ_MAX_GROUPED_DIM || K > DSMZ_MAX_GROUPED_DIM || N > DSMZ_MAX_GROUPED_DIM)
      return fail(DSMZ_ERR_UNSUPPORTED, me + "at most DSMZ_MAX_GROUPS groups and DSMZ_MAX_GROUPED_DIM rows or columns");
    if (flags & ~DSMZ_GROUPED_ACCUMULATE) return fail(DSMZ_ERR_INVALID, me + "unknown flag");
    if (!out || (M > 0 && (!x || !dy || !row_offsets))) return fail(DSMZ_ERR_INVALID, me + "null pointer");
    if (!aligned(out, 4) || !aligned(row_offsets, 4)) return fail(DSMZ_ERR_INVALID, me + "a pointer is not aligned to its type");
    if (!std::isfinite(alpha)) return fail(DSMZ_ERR_INVALID, me + "alpha must be finite");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M == 0) {
      if (flags & DSMZ_GROUPED_ACCUMULATE) return DSMZ_OK;
      cudaError_t e = cudaMemsetAsync(out, 0, static_cast<size_t>(G) * K * N * sizeof(float), s);
      return e == cudaSuccess ? DSMZ_OK : cuda_fail("dsmz_grouped_weight_grad", e);
    }
    if (ld_x < K || ld_dy < N || ld_x > kMaxElems || ld_dy > kMaxElems)
      return fail(DSMZ_ERR_INVALID, me + "a pitch is smaller than its row, or out of range");
    if (!aligned(x, 16) || !aligned(dy, 16) || ld_x % 8 || ld_dy % 8)
      return fail(DSMZ_ERR_INVALID, me + "x and dy need 16-byte aligned bases and pitches that are multiples of 8 elements");
    const int64_t nout = static_cast<int64_t>(G) * K * N * 4;
    if (overlaps(out, nout, x, ((M - 1) * ld_x + K) * 2) || overlaps(out, nout, dy, ((M - 1) * ld_dy + N) * 2))
      return fail(DSMZ_ERR_INVALID, me + "out overlaps an operand");
    int sms = 0, rc = sm_count(&sms);
    if (rc) return rc;
    const bool xw = K >= N;                              // the wider operand gives the tile's 128 rows
    const int64_t wide = xw ? K : N, narrow = xw ? N : K;
    gr::Args a{};
    a.offsets = row_offsets;
    a.G = G;
    a.M = M;
    a.mdim = static_cast<int32_t>(wide);
    a.ndim = static_cast<int32_t>(narrow);
    a.out = out;
    a.ld = N;
    a.gstride = K * N;
    a.transposed = xw ? 0 : 1;
    a.out_f32 = 1;
    a.accumulate = (flags & DSMZ_GROUPED_ACCUMULATE) ? 1 : 0;
    a.vec = aligned(out, 16) && N % 4 == 0;
    a.alpha = alpha;
    a.chunk = gr::kChunk;
    a.mtn = static_cast<int32_t>((wide + gr::kBM - 1) / gr::kBM);
    const int bnt = columns_for(narrow, static_cast<int64_t>(G) * a.mtn, sms);
    a.bn = static_cast<int32_t>(narrow >= bnt ? bnt : (narrow + 15) / 16 * 16);
    a.ntn = static_cast<int32_t>((narrow + a.bn - 1) / a.bn);
    const int64_t tiles = static_cast<int64_t>(G) * a.mtn * a.ntn;
    if (tiles > (1 << 27)) return fail(DSMZ_ERR_UNSUPPORTED, me + "too many tiles");
    const int64_t nk = (M / G + gr::kBK - 1) / gr::kBK;
    a.split = split_for(bnt, tiles, nk);
    CUtensorMap A, B, C{};
    if (!encode_width(&A, &a.a_slabs, xw ? x : dy, wide, M, xw ? ld_x : ld_dy, gr::kBM) ||
        !encode_width(&B, &a.b_slabs, xw ? dy : x, narrow, M, xw ? ld_dy : ld_x, a.bn))
      return fail(DSMZ_ERR_CUDA, me + "the driver refused a tensor map");
    if (a.vec && !a.accumulate && !a.transposed && a.split == 1) {
      const uint64_t dc[3] = {static_cast<uint64_t>(N), static_cast<uint64_t>(K), static_cast<uint64_t>(G)};
      const uint64_t sc[2] = {static_cast<uint64_t>(N) * 4, static_cast<uint64_t>(K) * N * 4};
      a.tma_out = encode_map(&C, out, 3, dc, sc, 32, 32, true);
    }
    return launch_grouped_bn<1, true>(bnt, a, A, B, C, tiles, nk, sms, "dsmz_grouped_weight_grad", s);
  });
}

int dsmz_first_order_set_wait_limit(int64_t ns) {
  if (ns < 0 || ns > int64_t{60} * 1000000000)
    return fail(DSMZ_ERR_INVALID, "dsmz_first_order_set_wait_limit: 0 to 60 s");
  g_wait_ns.store(ns, std::memory_order_relaxed);
  return DSMZ_OK;
}

int32_t dsmz_first_order_device_error(dsmz_stream_t stream) {
  int v = -1, zero = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cudaMemcpyFromSymbolAsync(&v, g_wait_err, sizeof(v), 0, cudaMemcpyDeviceToHost, s) != cudaSuccess ||
      cudaStreamSynchronize(s) != cudaSuccess)
    return -1;
  if (v != 0) {
    cudaMemcpyToSymbolAsync(g_wait_err, &zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
    cudaStreamSynchronize(s);
  }
  return v;
}

size_t dsmz_contrastive_loss_grad_workspace_bytes(int64_t ntok) {
  return ntok > 0 ? static_cast<size_t>(ntok) * sizeof(double) : sizeof(double);
}

int dsmz_contrastive_loss_grad(int32_t kind, const void* logits, int64_t V, int64_t ld, const int32_t* targets,
                               int64_t ntok, const int64_t* seq_start, const double* advantages, int32_t nseq,
                               double grad_scale, float* loss, void* grad, int64_t ld_grad, void* workspace,
                               size_t workspace_bytes, dsmz_stream_t stream) {
  return guarded("dsmz_contrastive_loss_grad", [&]() -> int {
    const std::string me = "dsmz_contrastive_loss_grad: ";
    if (!logits || !targets || !seq_start || !advantages || !loss || !grad || !workspace)
      return fail(DSMZ_ERR_INVALID, me + "null pointer");
    if (kind != DSMZ_SCORE_LOGITS_F32 && kind != DSMZ_SCORE_LOGITS_BF16)
      return fail(DSMZ_ERR_INVALID, me + "kind must be DSMZ_SCORE_LOGITS_F32 or DSMZ_SCORE_LOGITS_BF16");
    if (nseq < 1 || nseq > sg::kMaxSeqs)
      return fail(DSMZ_ERR_INVALID, me + "1 <= nseq <= " + std::to_string(sg::kMaxSeqs));
    if (V < 1 || V > 0x7fffffff || ld < V || ld_grad < V || ld > kMaxElems || ld_grad > kMaxElems)
      return fail(DSMZ_ERR_INVALID, me + "need 1 <= V < 2^31, ld >= V and ld_grad >= V");
    if (ntok < 1 || ntok > 0x7fffffff || seq_start[0] != 0 || seq_start[nseq] != ntok)
      return fail(DSMZ_ERR_INVALID, me + "seq_start must run from 0 to ntok >= 1");
    if (!std::isfinite(grad_scale)) return fail(DSMZ_ERR_INVALID, me + "grad_scale must be finite");
    const int64_t es = kind == DSMZ_SCORE_LOGITS_F32 ? 4 : 2;
    if (!aligned(logits, es) || !aligned(grad, es) || !aligned(targets, 4) || !aligned(loss, 4))
      return fail(DSMZ_ERR_INVALID, me + "a pointer is not aligned to its element type");
    if (rows_meet(logits, V * es, ld * es, grad, V * es, ld_grad * es, ntok) && !(logits == grad && (ld == ld_grad || ntok == 1)))
      return fail(DSMZ_ERR_INVALID, me + "the gradient may overwrite the logits in place, not overlap them otherwise");
    sg::Seqs q{};
    q.n = nseq;
    for (int i = 0; i < nseq; ++i) {
      const int64_t len = seq_start[i + 1] - seq_start[i];
      // the reference's mean over a sequence (ds_mezo/controller.py:14-15) has no empty case
      if (len < 1) return fail(DSMZ_ERR_INVALID, me + "every sequence needs a scored token");
      q.start[i] = seq_start[i];
      q.w[i] = advantages[i] / static_cast<double>(len);
    }
    q.start[nseq] = ntok;
    if (workspace_bytes < dsmz_contrastive_loss_grad_workspace_bytes(ntok) || !aligned(workspace, 8))
      return fail(DSMZ_ERR_WORKSPACE, me + "workspace too small or not 8-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* term = static_cast<double*>(workspace);
    return kind == DSMZ_SCORE_LOGITS_F32
               ? loss_grad<float>(logits, V, ld, targets, ntok, q, grad_scale, loss, grad, ld_grad, term, s)
               : loss_grad<__nv_bfloat16>(logits, V, ld, targets, ntok, q, grad_scale, loss, grad, ld_grad, term, s);
  });
}

int dsmz_adamw_step(const dsmz_adamw_desc* desc, const dsmz_adamw_tensor* tensors, int32_t n, void* workspace,
                    size_t workspace_bytes, dsmz_stream_t stream) {
  return guarded("dsmz_adamw_step", [&]() -> int {
    if (!desc) return fail(DSMZ_ERR_INVALID, "dsmz_adamw_step: null descriptor");
    const dsmz_adamw_desc& d = *desc;
    if ((d.param_dtype != DSMZ_F32 && d.param_dtype != DSMZ_BF16) || (d.grad_dtype != DSMZ_F32 && d.grad_dtype != DSMZ_BF16))
      return fail(DSMZ_ERR_INVALID, "dsmz_adamw_step: parameters and gradients must be DSMZ_F32 or DSMZ_BF16");
    if (d.state_bits != 32 && d.state_bits != 8) return fail(DSMZ_ERR_INVALID, "dsmz_adamw_step: state_bits must be 32 or 8");
    if (!(d.beta1 >= 0.0 && d.beta1 < 1.0 && d.beta2 >= 0.0 && d.beta2 < 1.0) || !(d.eps >= 0.0) || !(d.weight_decay >= 0.0) ||
        !std::isfinite(d.eps) || !std::isfinite(d.weight_decay) || (!d.lr_device && !std::isfinite(d.lr)))
      return fail(DSMZ_ERR_INVALID, "dsmz_adamw_step: need 0 <= beta < 1, eps >= 0, weight_decay >= 0 and a finite lr");
    if (d.state_bits == 8 && d.eps < 1e-12)
      return fail(DSMZ_ERR_INVALID, "dsmz_adamw_step: 8-bit states need eps >= 1e-12 (their denominators drop v below 2^-126)");
    if (!d.step_counter && d.step < 1) return fail(DSMZ_ERR_INVALID, "dsmz_adamw_step: steps count from 1");
    int rc = check_tensors("dsmz_adamw_step", tensors, n, d.state_bits, false, d.param_dtype, d.grad_dtype);
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    aw::Coef c{};
    aw::Coef* dc = nullptr;
    if (d.step_counter || d.lr_device) {
      if (!workspace || workspace_bytes < DSMZ_ADAMW_WORKSPACE_BYTES || !aligned(workspace, 16))
        return fail(DSMZ_ERR_WORKSPACE, "dsmz_adamw_step: a device counter or lr needs a 16-byte aligned workspace of "
                                        "DSMZ_ADAMW_WORKSPACE_BYTES");
      dc = static_cast<aw::Coef*>(workspace);
      aw::k_adamw_coef<<<1, 1, 0, s>>>(d.step_counter, d.lr_device, d.lr, d.weight_decay, d.beta1, d.beta2, d.step, dc);
      DSMZ_LAUNCHED("dsmz_adamw_step: coefficients");
    } else {
      const double t = static_cast<double>(d.step);
      c.decay = static_cast<float>(1.0 - d.lr * d.weight_decay);
      c.inv_root = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(d.beta2, t)));
      c.step = static_cast<float>(d.lr / (1.0 - std::pow(d.beta1, t)));
    }
    return n <= kSmall ? adamw_run<kSmall>(d, tensors, n, c, dc, s) : adamw_run<kLarge>(d, tensors, n, c, dc, s);
  });
}

int dsmz_adamw_state_values(const dsmz_adamw_tensor* tensors, int32_t n, dsmz_stream_t stream) {
  return guarded("dsmz_adamw_state_values", [&]() -> int {
    int rc = check_tensors("dsmz_adamw_state_values", tensors, n, 8, true, DSMZ_F32, DSMZ_F32);
    if (rc) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return n <= kSmall ? adamw_values<kSmall>(tensors, n, s) : adamw_values<kLarge>(tensors, n, s);
  });
}

}  // extern "C"
