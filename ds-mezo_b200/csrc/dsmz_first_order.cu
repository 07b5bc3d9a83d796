// C ABI of the first-order operators declared in dsmezo.h: the scoring loss with its gradient
// and AdamW over many tensors.
#include <cmath>
#include <exception>
#include <vector>

#include "dsmezo.h"
#include "dsmz_adamw.cuh"
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
int chunked(const dsmz_adamw_tensor* tensors, int32_t n, const char* what, Fill fill, Launch launch) {
  auto box = std::vector<aw::Args<CAP>>(1);
  aw::Args<CAP>& a = box[0];
  int32_t i = 0;
  while (i < n) {
    a.n = 0;
    int64_t tiles = 0;
    for (; i < n && a.n < CAP; ++i) {
      if (tensors[i].n == 0) continue;
      const int64_t nt = (tensors[i].n + aw::kTile - 1) / aw::kTile;
      if (tiles + nt > 0x7fffffff) {
        if (a.n > 0) break;
        return fail(DSMZ_ERR_UNSUPPORTED, std::string(what) + ": a tensor of more than 2^42 elements");
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
      tensors, n, "dsmz_adamw_state_values",
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
      tensors, n, "dsmz_adamw_step",
      [&](aw::Args<CAP>& a, int k, const dsmz_adamw_tensor& t) {
        a.b1 = d.beta1; a.omb1 = 1.0 - d.beta1;
        a.b2 = d.beta2; a.omb2 = 1.0 - d.beta2;
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
  sg::k_loss_sum<<<1, 256, 0, s>>>(term, ntok, loss);
  DSMZ_LAUNCHED("dsmz_contrastive_loss_grad: sum");
  return DSMZ_OK;
}

}  // namespace

extern "C" {

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
    const uintptr_t a = reinterpret_cast<uintptr_t>(logits), b = reinterpret_cast<uintptr_t>(grad);
    const uintptr_t na = static_cast<uintptr_t>(((ntok - 1) * ld + V) * es), nb = static_cast<uintptr_t>(((ntok - 1) * ld_grad + V) * es);
    if (a < b + nb && b < a + na && !(a == b && (ld == ld_grad || ntok == 1)))
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
