// What the gradient norm (grad_norm.hip) leaves for the kernels that scale by it (grad_scale, the clipped Adam step).
#pragma once
#include "common.h"

namespace pr {

constexpr int NORM_SETS = 32;       // norms a call takes at once

// Partials of a set that every workgroup of the kernel after the norm adds itself; more are added by a kernel in between.
// The scaling has up to 2048 workgroups, for which eight loads a thread are less than a launch (a scene of 1 M Gaussians
// 290 against 293 us, 56 ragged tensors 49 against 52); the Adam step has one for 4096 elements, so they are worth it where one load a thread does.
constexpr unsigned SCALE_JOINS = 2304, ADAM_JOINS = 256;

// Partials of set s: [first[s], first[s + 1]) of `partials`; one only (its total) where a kernel has added them.
struct NormSets {
  const double *partials;
  unsigned first[NORM_SETS + 1];
};

template <int KIND>
__device__ __forceinline__ double norm_combine(double a, double b) {
  if (KIND != PR_NORM_INF) return a + b;
  return (a > b || a != a) ? a : b;  // max that keeps NaN
}

// Over the 256 threads of a workgroup.
template <int KIND>
__device__ __forceinline__ double norm_block_combine(double v) {
  __shared__ double part[4];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = norm_combine<KIND>(v, __shfl_xor(v, d));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) v = norm_combine<KIND>(v, part[i]);
  return v;
}

// The norm of set s, the same for every workgroup that asks: partials are added in one order.
template <int KIND>
__device__ __forceinline__ double norm_of_set(const NormSets &n, int s) {
  double v = 0.;
  for (unsigned i = n.first[s] + threadIdx.x; i < n.first[s + 1]; i += 256) v = norm_combine<KIND>(v, n.partials[i]);
  v = norm_block_combine<KIND>(v);
  return KIND == PR_NORM_2 ? sqrt(v) : v;
}

// Factor that brings gradients of this norm to at most max_norm, as torch.nn.utils.clip_grad_norm_ forms it, rounded
// once: a norm within bounds gives exactly 1, a NaN norm NaN.
__device__ __forceinline__ float clip_coefficient(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  return c >= 1. ? 1.f : (float)c;
}

int check_grad_tensors(const pr_grad_tensor *tensors, int n, int n_sets);
size_t grad_norm_scratch(const pr_grad_tensor *tensors, int n);
// A set without elements has no workgroup that would write its norm (0): writes them all then.
int write_empty_norms(const pr_grad_tensor *tensors, int n, int n_sets, void *scratch, size_t scratch_bytes, float *norms,
                      void *stream);
// Norm kernels of the tensors, ordered by set; on return `sets` says where each set's partials are, at most `joins`.
int launch_grad_norms(const pr_grad_tensor *tensors, int n, int n_sets, int kind, unsigned joins, void *scratch,
                      size_t scratch_bytes, NormSets *sets, hipStream_t st);

}  // namespace pr
