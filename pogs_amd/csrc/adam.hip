// Fused multi-group Adam step (pr_adam_step): every parameter group that is due this iteration is updated
// in ONE launch.
//
// Replaces the per-group `torch.optim.Adam(...).step()` calls the trainer issues through
// nerfstudio's Optimizers.optimizer_scaler_step_some (nerfstudio/engine/optimizers.py:159-172, driven by
// nerfstudio/engine/trainer.py:494-510) with the groups, learning rates and eps of pogs/pogs_config.py:38-85.
// The arithmetic is torch.optim.Adam's single-tensor update (betas, eps, no weight decay, no amsgrad,
// maximize=False), in its order of operations:
//   m  = m + (g - m)(1 - beta1)                       exp_avg.lerp_(grad, 1 - beta1)
//   v  = v beta2 + (1 - beta2) g g                     exp_avg_sq.mul_(beta2).addcmul_(grad, grad, 1 - beta2)
//   p -= (lr / (1 - beta1^t)) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// The host passes lr / (1 - beta1^t) and sqrt(1 - beta2^t) per group (computed in double, as torch does).
//
// HBM-bound streaming kernel: 16 B read + 12 B written per element.  Workgroups are assigned to
// (group, chunk) pairs through a prefix table in the kernel argument, so small and large groups share one
// grid; each lane handles four consecutive elements with 16-byte accesses.
#include <math.h>

#include <stdlib.h>

#include "grad_norm.h"

namespace pr {
namespace {

constexpr int MAX_GROUPS = 16;
constexpr int BLOCK = 256;
constexpr int PER_BLOCK = BLOCK * 4 * 4;  // elements per workgroup: 4 float4 per lane

struct AdamTable {
  float *param[MAX_GROUPS];
  const float *grad[MAX_GROUPS];
  float *exp_avg[MAX_GROUPS];
  float *exp_avg_sq[MAX_GROUPS];
  int64_t numel[MAX_GROUPS];
  float step_size[MAX_GROUPS], one_minus_beta1[MAX_GROUPS], beta2[MAX_GROUPS], one_minus_beta2[MAX_GROUPS],
      bias2_sqrt[MAX_GROUPS], eps[MAX_GROUPS];
  unsigned first_block[MAX_GROUPS + 1];
  int n;
};
struct ClipTable {  // per group: the set whose norm its gradient is clipped by (-1: not clipped) and what it may be
  NormSets sets;
  int set[MAX_GROUPS];
  double max_norm[MAX_GROUPS];
  float *norms;
};
struct NoClip {};
// From the last element to the first where a norm has been taken just before: the end of the gradients is still cached.
__device__ __forceinline__ unsigned block_of(const NoClip &) { return blockIdx.x; }
__device__ __forceinline__ unsigned block_of(const ClipTable &) { return gridDim.x - 1 - blockIdx.x; }
__device__ __forceinline__ float gradient_factor(const NoClip &, int, bool) { return 1.f; }
__device__ __forceinline__ float gradient_factor(const ClipTable &c, int gi, bool first) {
  const int s = c.set[gi];
  if (s < 0) return 1.f;
  const double norm = norm_of_set<PR_NORM_2>(c.sets, s);
  if (first && threadIdx.x == 0) c.norms[s] = (float)norm;   // (every group of the set writes the same)
  return clip_coefficient(norm, c.max_norm[gi]);
}

__device__ __forceinline__ void adam_update(float &p, float g, float &m, float &v, float step_size, float omb1,
                                            float beta2, float omb2, float bias2_sqrt, float eps) {
  m = m + (g - m) * omb1;
  v = v * beta2 + omb2 * g * g;
  const float denom = sqrtf(v) / bias2_sqrt + eps;
  p = p - step_size * (m / denom);
}

// CLIP = ClipTable: every gradient is taken times its group's factor, which is the same for all of a workgroup's
// elements.  CLIP = NoClip: the factor is a constant 1 and drops out.
template <typename CLIP>
__global__ void __launch_bounds__(BLOCK) adam_kernel(const AdamTable t, const CLIP clip) {
  const unsigned block = block_of(clip);
  int gi = 0;
#pragma unroll 1
  while (gi + 1 < t.n && block >= t.first_block[gi + 1]) ++gi;
  const int64_t n = t.numel[gi];
  float *__restrict__ p = t.param[gi];
  const float *__restrict__ g = t.grad[gi];
  float *__restrict__ m = t.exp_avg[gi];
  float *__restrict__ v = t.exp_avg_sq[gi];
  const float ss = t.step_size[gi], omb1 = t.one_minus_beta1[gi], b2 = t.beta2[gi], omb2 = t.one_minus_beta2[gi],
              bc = t.bias2_sqrt[gi], eps = t.eps[gi];
  const int64_t base = (int64_t)(block - t.first_block[gi]) * PER_BLOCK;
  const float factor = gradient_factor(clip, gi, base == 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int64_t i = base + ((int64_t)r * BLOCK + threadIdx.x) * 4;
    if (i + 3 < n) {
      float4 pp = *reinterpret_cast<float4 *>(p + i), mm = *reinterpret_cast<float4 *>(m + i);
      float4 vv = *reinterpret_cast<float4 *>(v + i);
      float4 gg = *reinterpret_cast<const float4 *>(g + i);
      gg.x *= factor, gg.y *= factor, gg.z *= factor, gg.w *= factor;
      adam_update(pp.x, gg.x, mm.x, vv.x, ss, omb1, b2, omb2, bc, eps);
      adam_update(pp.y, gg.y, mm.y, vv.y, ss, omb1, b2, omb2, bc, eps);
      adam_update(pp.z, gg.z, mm.z, vv.z, ss, omb1, b2, omb2, bc, eps);
      adam_update(pp.w, gg.w, mm.w, vv.w, ss, omb1, b2, omb2, bc, eps);
      *reinterpret_cast<float4 *>(p + i) = pp;
      *reinterpret_cast<float4 *>(m + i) = mm;
      *reinterpret_cast<float4 *>(v + i) = vv;
    } else {
      for (int64_t k = i; k < n; ++k) {
        float pk = p[k], mk = m[k], vk = v[k];
        adam_update(pk, g[k] * factor, mk, vk, ss, omb1, b2, omb2, bc, eps);
        p[k] = pk;
        m[k] = mk;
        v[k] = vk;
      }
    }
  }
}

}  // namespace
}  // namespace pr

extern "C" int pr_adam_max_groups(void) { return pr::MAX_GROUPS; }

namespace pr {
namespace {
int check_groups(const pr_adam_group *groups, int n_groups) {
  for (int i = 0; i < n_groups; ++i) {
    const pr_adam_group &g = groups[i];
    if (g.numel < 0 || g.step < 1 || !(g.beta1 >= 0.0 && g.beta1 < 1.0) || !(g.beta2 >= 0.0 && g.beta2 < 1.0))
      return PR_EINVAL;
    if (g.numel == 0) continue;
    if (!g.param || !g.grad || !g.exp_avg || !g.exp_avg_sq) return PR_EINVAL;
    // 16-byte accesses: torch allocations are; a sliced view might not be
    if ((((uintptr_t)g.param | (uintptr_t)g.grad | (uintptr_t)g.exp_avg | (uintptr_t)g.exp_avg_sq) & 15) != 0)
      return PR_EINVAL;
  }
  return PR_OK;
}

// Arguments checked.  clips and sets NULL: not clipped.
int adam_launch(const pr_adam_group *groups, const pr_clip_rule *clips, const NormSets *sets, float *norms, int n_groups,
                hipStream_t st) {
  AdamTable t;
  ClipTable c;
  t.n = 0;
  unsigned blocks = 0;
  for (int i = 0; i < n_groups; ++i) {
    const pr_adam_group &g = groups[i];
    if (g.numel == 0) continue;
    const int k = t.n++;
    c.set[k] = clips ? clips[i].set : -1;
    c.max_norm[k] = clips ? clips[i].max_norm : 0.;
    t.param[k] = g.param;
    t.grad[k] = g.grad;
    t.exp_avg[k] = g.exp_avg;
    t.exp_avg_sq[k] = g.exp_avg_sq;
    t.numel[k] = g.numel;
    // scalars are formed in double and rounded once, as torch does with its Python-float hyperparameters
    const double bias1 = 1.0 - pow(g.beta1, (double)g.step);
    const double bias2 = 1.0 - pow(g.beta2, (double)g.step);
    t.step_size[k] = (float)(g.lr / bias1);
    t.one_minus_beta1[k] = (float)(1.0 - g.beta1);
    t.beta2[k] = (float)g.beta2;
    t.one_minus_beta2[k] = (float)(1.0 - g.beta2);
    t.bias2_sqrt[k] = (float)sqrt(bias2);
    t.eps[k] = (float)g.eps;
    t.first_block[k] = blocks;
    const int64_t nb = (g.numel + PER_BLOCK - 1) / PER_BLOCK;
    if (nb + blocks > 0x7fffffffll) return PR_EUNSUPPORTED;
    blocks += (unsigned)nb;
  }
  if (t.n == 0) return PR_OK;
  t.first_block[t.n] = blocks;
  if (!clips) {
    hipLaunchKernelGGL(adam_kernel<NoClip>, dim3(blocks), dim3(BLOCK), 0, st, t, NoClip{});
    return check_launch("pr_adam_step");
  }
  c.sets = *sets;
  c.norms = norms;
  hipLaunchKernelGGL(adam_kernel<ClipTable>, dim3(blocks), dim3(BLOCK), 0, st, t, c);
  return check_launch("pr_adam_step_clipped");
}

// The clipped groups' gradients as tensors, ordered by set; -1 where the arguments are not valid.
int clipped_tensors(const pr_adam_group *groups, const pr_clip_rule *clips, int n_groups, int n_sets, pr_grad_tensor *out) {
  int m = 0;
  for (int i = 0; i < n_groups; ++i) {
    if (clips[i].set < 0) continue;
    if (!(clips[i].max_norm >= 0.0)) return -1;
    out[m++] = pr_grad_tensor{const_cast<float *>(groups[i].grad), groups[i].numel, PR_F32, clips[i].set};
  }
  return check_grad_tensors(out, m, n_sets) == PR_OK ? m : -1;
}

struct Tensors {  // freed at the end of a call
  pr_grad_tensor *p;
  explicit Tensors(int n) : p((pr_grad_tensor *)malloc(sizeof(pr_grad_tensor) * (size_t)(n > 0 ? n : 1))) {}
  ~Tensors() { free(p); }
};
}  // namespace
}  // namespace pr

extern "C" int pr_adam_step(const pr_adam_group *groups, int n_groups, void *stream) {
  if (n_groups < 0 || n_groups > pr::MAX_GROUPS) return PR_EINVAL;
  if (n_groups == 0) return PR_OK;
  if (!groups) return PR_EINVAL;
  const int rc = pr::check_groups(groups, n_groups);
  if (rc != PR_OK) return rc;
  return pr::adam_launch(groups, nullptr, nullptr, nullptr, n_groups, (hipStream_t)stream);
}

extern "C" size_t pr_adam_clip_scratch_bytes(const pr_adam_group *groups, const pr_clip_rule *clips, int n_groups, int n_sets) {
  if (n_groups < 0 || !groups || !clips) return 0;
  pr::Tensors t(n_groups);
  if (!t.p) return 0;
  const int n = pr::clipped_tensors(groups, clips, n_groups, n_sets, t.p);
  return n < 0 ? 0 : pr::grad_norm_scratch(t.p, n);
}

extern "C" int pr_adam_step_clipped(const pr_adam_group *groups, const pr_clip_rule *clips, int n_groups, int n_sets,
                                    void *scratch, size_t scratch_bytes, float *norms, void *stream) {
  if (n_groups < 0) return PR_EINVAL;
  if (n_groups == 0) return PR_OK;
  if (!groups || !clips || !scratch || ((uintptr_t)scratch & 7) || !norms) return PR_EINVAL;
  pr::Tensors t(n_groups);
  if (!t.p) return PR_ESCRATCH;
  const int n = pr::clipped_tensors(groups, clips, n_groups, n_sets, t.p);
  if (n < 0) return PR_EINVAL;
  if (scratch_bytes < pr::grad_norm_scratch(t.p, n)) return PR_ESCRATCH;
  hipStream_t st = (hipStream_t)stream;
  pr::NormSets sets;
  int rc = pr::check_groups(groups, n_groups);
  if (rc != PR_OK) return rc;
  rc = pr::write_empty_norms(t.p, n, n_sets, scratch, scratch_bytes, norms, stream);
  if (rc != PR_OK) return rc;
  rc = pr::launch_grad_norms(t.p, n, n_sets, PR_NORM_2, pr::ADAM_JOINS, scratch, scratch_bytes, &sets, st);
  for (int i = 0; rc == PR_OK && i < n_groups; i += pr::MAX_GROUPS)
    rc = pr::adam_launch(groups + i, clips + i, &sets, norms, n_groups - i < pr::MAX_GROUPS ? n_groups - i : pr::MAX_GROUPS, st);
  return rc;
}
