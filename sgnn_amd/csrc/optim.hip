// Fused Adam over the flat fp32 parameter buffer (replaces torch.optim.Adam's
// multi-tensor path used by sgnn/single_scale/train.py:199,271-273).
// Same arithmetic order as torch 2.x Adam (amsgrad=False, weight_decay=0):
//   m = lerp(m, g, 1-b1) ; v = v*b2 + (1-b2)*g*g
//   p += -step_size * m / (sqrt(v)/sqrt(1-b2^t) + eps),  step_size = lr/(1-b1^t)
#include "common.h"
#include "../../include/sgnn.h"
#include "sgnn_internal.h"

namespace {
// One Adam element, in torch's order of operations.
SGNN_DEV void adam_element(float* p, float gi, float* m, float* v, float w1, float b2, float omb2, float neg_step,
                           float bc2_sqrt, float eps) {
  float mi = *m;
  mi = __fadd_rn(mi, __fmul_rn(w1, __fsub_rn(gi, mi)));  // lerp, weight < 0.5 branch
  const float vi = __fadd_rn(__fmul_rn(*v, b2), __fmul_rn(omb2, __fmul_rn(gi, gi)));
  const float denom = __fadd_rn(__fdiv_rn(sqrtf(vi), bc2_sqrt), eps);
  *p = __fadd_rn(*p, __fmul_rn(neg_step, __fdiv_rn(mi, denom)));
  *m = mi;
  *v = vi;
}

__global__ __launch_bounds__(256) void k_adam(float* __restrict__ p, const float* __restrict__ g,
                                              float* __restrict__ m, float* __restrict__ v,
                                              int64_t n, float w1, float b2, float omb2,
                                              float neg_step, float bc2_sqrt, float eps) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x) {
    adam_element(p + i, g[i], m + i, v + i, w1, b2, omb2, neg_step, bc2_sqrt, eps);
  }
}

// Workgroups (x, segment): the moments of the matrices and the whole step of the other parameters (include/sgnn.h,
// sgnn_muon_moments); bounded by memory, one launch for all parameters of a model.
__global__ __launch_bounds__(256) void k_muon_moments(const sgnn_muon_seg* segs, float* param, const float* grad,
                                                      float* m, float* v, float* update, float momentum, int nesterov,
                                                      float w1, float b2, float omb2, float neg_step, float bc2_sqrt,
                                                      float eps) {
  const sgnn_muon_seg s = segs[blockIdx.y];
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < s.numel; t += (int64_t)gridDim.x * 256) {
    const int64_t i = s.offset + t;
    const float g = grad[i];
    if (s.matrix) {
      const float b = momentum * m[i] + g;
      m[i] = b;
      update[i] = nesterov ? g + momentum * b : b;
    } else {
      adam_element(param + i, g, m + i, v + i, w1, b2, omb2, neg_step, bc2_sqrt, eps);
    }
  }
}

__global__ __launch_bounds__(256) void k_muon_apply(const sgnn_muon_seg* segs, float* param, const float* update,
                                                    float lr, float keep) {
  const sgnn_muon_seg s = segs[blockIdx.y];
  if (!s.matrix) return;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < s.numel; t += (int64_t)gridDim.x * 256)
    param[s.offset + t] = keep * param[s.offset + t] - lr * s.scale * update[s.offset + t];
}

constexpr unsigned kMuonBlocks = 32;  // per segment: 8192 elements at a time, grid-strided past them
}  // namespace

extern "C" int sgnn_adam_step(float* param, const float* grad, float* exp_avg, float* exp_avg_sq,
                              int64_t n, float lr, float beta1, float beta2, float eps,
                              int64_t step, void* stream) {
  using namespace sgnn;
  if (!param || !grad || !exp_avg || !exp_avg_sq || n < 0 || step < 1)
    return set_error(SGNN_ERR_INVALID, "adam_step: bad arguments");
  if (!(1.0f - beta1 < 0.5f)) return set_error(SGNN_ERR_UNSUPPORTED, "adam_step: beta1 <= 0.5");
  const double bc1 = 1.0 - pow((double)beta1, (double)step);
  const double bc2 = 1.0 - pow((double)beta2, (double)step);
  const float neg_step = (float)(-(double)lr / bc1);
  const float bc2_sqrt = (float)sqrt(bc2);
  const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 2048);
  if (n == 0) return SGNN_OK;
  hipLaunchKernelGGL(k_adam, dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream), param,
                     grad, exp_avg, exp_avg_sq, n, 1.0f - beta1, beta2, 1.0f - beta2, neg_step,
                     bc2_sqrt, eps);
  return check_launch("adam_step");
}

extern "C" int sgnn_muon_moments(const sgnn_muon_seg* segs, int32_t nseg, float* param, const float* grad, float* m,
                                 float* v, float* update, float momentum, int32_t nesterov, float adam_lr, float beta1,
                                 float beta2, float adam_eps, int64_t step, void* stream) {
  using namespace sgnn;
  if (nseg < 0 || nseg > 65535 || (nseg > 0 && (!segs || !param || !grad || !m || !v || !update)) || step < 1)
    return set_error(SGNN_ERR_INVALID, "muon_moments: bad arguments");
  if (!(1.0f - beta1 < 0.5f)) return set_error(SGNN_ERR_UNSUPPORTED, "muon_moments: beta1 <= 0.5");
  if (nseg == 0) return SGNN_OK;
  const double bc1 = 1.0 - pow((double)beta1, (double)step), bc2 = 1.0 - pow((double)beta2, (double)step);
  hipLaunchKernelGGL(k_muon_moments, dim3(kMuonBlocks, (unsigned)nseg), dim3(256), 0, static_cast<hipStream_t>(stream),
                     segs, param, grad, m, v, update, momentum, nesterov ? 1 : 0, 1.0f - beta1, beta2, 1.0f - beta2,
                     (float)(-(double)adam_lr / bc1), (float)sqrt(bc2), adam_eps);
  return check_launch("muon_moments");
}

extern "C" int sgnn_muon_apply(const sgnn_muon_seg* segs, int32_t nseg, float* param, const float* update, float lr,
                               float weight_decay, void* stream) {
  using namespace sgnn;
  if (nseg < 0 || nseg > 65535 || (nseg > 0 && (!segs || !param || !update)))
    return set_error(SGNN_ERR_INVALID, "muon_apply: bad arguments");
  if (nseg == 0) return SGNN_OK;
  hipLaunchKernelGGL(k_muon_apply, dim3(kMuonBlocks, (unsigned)nseg), dim3(256), 0, static_cast<hipStream_t>(stream),
                     segs, param, update, lr, 1.0f - lr * weight_decay);
  return check_launch("muon_apply");
}
