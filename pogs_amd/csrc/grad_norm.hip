// Norm of the gradients of many tensors and their scaling to at most a given norm (pr_grad_norm / pr_grad_clip).
//
// Stands in for torch.nn.utils.clip_grad_norm_, which nerfstudio's Optimizers.optimizer_scaler_step_some calls for every
// parameter group with a max_norm (nerfstudio/engine/optimizers.py:159-172).
//   norm_s = sqrt(sum over the tensors of set s of g^2)        (or sum |g|, or max |g|)
//   g     <- g * min(1, max_norm_s / (norm_s + 1e-6))
//
// HBM-bound: the norm reads every gradient once, the scaling reads and writes it once.  Every tensor of a launch gets
// workgroups by its size, at least one (a workgroup that went through several small tensors would wait out the memory
// latency of each: 26 against 5 us for 56 tensors of 1 to 2 M elements), and they take its chunks of 4096 elements in
// turn, so that the chip reads one run of memory at a time.  The scaling goes through the chunks from the last to the
// first: the last ones read for the norm are still in the 256 MB cache behind HBM.  Sums are kept in float64 from the first
// element on (float32 gradients of 1e30 square to a finite value, and the order of the sum does not show in float32);
// partials go to memory, one per workgroup and set, and are added in one fixed order: the result does not depend on the
// order in which workgroups run.
#include <math.h>
#include <stdlib.h>

#include <algorithm>

#include "grad_norm.h"

namespace pr {
namespace {

constexpr int MAX_TENSORS = 128;  // per launch: the table travels in the kernel argument (at most 4 KB)
constexpr int BLOCK = 256;
constexpr int64_t CHUNK = 4096;  // elements a workgroup takes at a time: 16 each, in 16-byte accesses
constexpr int MAX_BLOCKS = 2048;  // per launch, besides one for each tensor: eight workgroups for each CU

struct Table {
  void *grad[MAX_TENSORS];
  int64_t numel[MAX_TENSORS];
  unsigned first_block[MAX_TENSORS + 1];
  unsigned char dtype[MAX_TENSORS], set[MAX_TENSORS];
  int n;
};

struct MaxNorms {
  double of[NORM_SETS];
};

__device__ __forceinline__ float from_bits16(unsigned short b, int dtype) {
  if (dtype == PR_F16) return (float)__builtin_bit_cast(_Float16, b);
  return __builtin_bit_cast(float, (unsigned)b << 16);
}
__device__ __forceinline__ unsigned short to_bits16(float v, int dtype) {
  if (dtype == PR_F16) return __builtin_bit_cast(unsigned short, (_Float16)v);
  return __builtin_bit_cast(unsigned short, (__bf16)v);
}

template <int KIND>
__device__ __forceinline__ void take(double &acc, float g) {
  if (KIND == PR_NORM_2) acc = fma((double)g, (double)g, acc);
  else acc = norm_combine<KIND>(acc, (double)fabsf(g));
}

// The tensor that a workgroup belongs to.
__device__ __forceinline__ int find_tensor(const Table &t, unsigned block) {
  int lo = 0, hi = t.n - 1;
#pragma unroll 1
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first_block[mid] <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// f(value) for this thread's elements of a chunk that starts at `lo` and has `left` elements (more than CHUNK: a whole one)
template <typename F>
__device__ __forceinline__ void each_of_chunk(const void *grad, int dtype, int64_t lo, int64_t left, F f) {
  if (dtype == PR_F32) {
    const float *g = (const float *)grad + lo;
    if (left >= CHUNK && aligned16(g)) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const float4 *>(g)[u * BLOCK + threadIdx.x];
#pragma unroll
      for (int u = 0; u < 4; ++u) f(v[u].x, 0), f(v[u].y, 1), f(v[u].z, 2), f(v[u].w, 3);
    } else {
#pragma unroll 8
      for (int u = 0; u < 16; ++u)
        if (u * BLOCK + (int)threadIdx.x < left) f(g[u * BLOCK + threadIdx.x], u & 3);
    }
  } else {
    const unsigned short *g = (const unsigned short *)grad + lo;
    if (left >= CHUNK && aligned16(g)) {
      uint4 v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = reinterpret_cast<const uint4 *>(g)[u * BLOCK + threadIdx.x];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const unsigned w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f(from_bits16((unsigned short)(w[k] & 0xffffu), dtype), k);
          f(from_bits16((unsigned short)(w[k] >> 16), dtype), k);
        }
      }
    } else {
#pragma unroll 8
      for (int u = 0; u < 16; ++u)
        if (u * BLOCK + (int)threadIdx.x < left) f(from_bits16(g[u * BLOCK + threadIdx.x], dtype), u & 3);
    }
  }
}

template <int KIND>
__global__ void __launch_bounds__(BLOCK) grad_norm_kernel(const Table t, double *__restrict__ partials) {
  const int k = find_tensor(t, blockIdx.x);
  const unsigned first = t.first_block[k], blocks = t.first_block[k + 1] - first;
  const int64_t n = t.numel[k];
  double acc[4] = {0., 0., 0., 0.};
  for (int64_t lo = (int64_t)(blockIdx.x - first) * CHUNK; lo < n; lo += (int64_t)blocks * CHUNK)
    each_of_chunk(t.grad[k], t.dtype[k], lo, n - lo, [&](float g, int at) { take<KIND>(acc[at], g); });
  const double all = norm_block_combine<KIND>(norm_combine<KIND>(norm_combine<KIND>(acc[0], acc[1]), norm_combine<KIND>(acc[2], acc[3])));
  if (threadIdx.x == 0) partials[blockIdx.x] = all;
}

// A workgroup a set: its total, and (totals NULL) its norm.
template <int KIND>
__global__ void __launch_bounds__(BLOCK) grad_norm_finish_kernel(const NormSets sets, double *__restrict__ totals,
                                                                 float *__restrict__ norms) {
  const int s = blockIdx.x;
  if (totals) {
    double v = 0.;
    for (unsigned i = sets.first[s] + threadIdx.x; i < sets.first[s + 1]; i += BLOCK) v = norm_combine<KIND>(v, sets.partials[i]);
    v = norm_block_combine<KIND>(v);
    if (threadIdx.x == 0) totals[s] = v;
  } else {
    const double norm = norm_of_set<KIND>(sets, s);
    if (threadIdx.x == 0) norms[s] = (float)norm;
  }
}

__device__ __forceinline__ void scale_chunk(void *grad, int dtype, int64_t lo, int64_t left, float c) {
  if (dtype == PR_F32) {
    float *g = (float *)grad + lo;
    if (left >= CHUNK && aligned16(g)) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<float4 *>(g)[u * BLOCK + threadIdx.x];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        reinterpret_cast<float4 *>(g)[u * BLOCK + threadIdx.x] = make_float4(v[u].x * c, v[u].y * c, v[u].z * c, v[u].w * c);
    } else {
#pragma unroll 8
      for (int u = 0; u < 16; ++u)
        if (u * BLOCK + (int)threadIdx.x < left) g[u * BLOCK + threadIdx.x] *= c;
    }
  } else {
    unsigned short *g = (unsigned short *)grad + lo;
    if (left >= CHUNK && aligned16(g)) {
      uint4 v[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) v[u] = reinterpret_cast<uint4 *>(g)[u * BLOCK + threadIdx.x];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        unsigned w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const unsigned a = to_bits16(from_bits16((unsigned short)(w[k] & 0xffffu), dtype) * c, dtype);
          const unsigned b = to_bits16(from_bits16((unsigned short)(w[k] >> 16), dtype) * c, dtype);
          w[k] = a | (b << 16);
        }
        reinterpret_cast<uint4 *>(g)[u * BLOCK + threadIdx.x] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll 8
      for (int u = 0; u < 16; ++u)
        if (u * BLOCK + (int)threadIdx.x < left)
          g[u * BLOCK + threadIdx.x] = to_bits16(from_bits16(g[u * BLOCK + threadIdx.x], dtype) * c, dtype);
    }
  }
}

template <int KIND>
__global__ void __launch_bounds__(BLOCK) grad_scale_kernel(const Table t, const NormSets sets, const MaxNorms max_norms,
                                                           float *__restrict__ norms) {
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const int k = find_tensor(t, block), set = t.set[k];
  const double norm = norm_of_set<KIND>(sets, set);
  const float c = clip_coefficient(norm, max_norms.of[set]);
  const unsigned first = t.first_block[k], blocks = t.first_block[k + 1] - first;
  if (block == first && threadIdx.x == 0) norms[set] = (float)norm;   // (every tensor of the set writes the same)
  // a norm within bounds leaves every value as it is: nothing to read or write (NaN is no such norm)
  if (c == 1.f) return;
  const int64_t n = t.numel[k], chunks = (n + CHUNK - 1) / CHUNK;
  // this workgroup's chunks, the last one first
  int64_t i = block - first;
  for (i += (chunks - 1 - i) / blocks * blocks; i >= 0; i -= blocks) scale_chunk(t.grad[k], t.dtype[k], i * CHUNK, n - i * CHUNK, c);
}

// Cuts the host's list into launches of at most MAX_TENSORS tensors.  next() fills the table (n == 0 at the end).
struct Launches {
  const pr_grad_tensor *tensors;
  int n, at = 0;
  Table t;
  unsigned blocks = 0;
  unsigned set_blocks[NORM_SETS];  // workgroups of each set in this launch
  Launches(const pr_grad_tensor *tensors_, int n_) : tensors(tensors_), n(n_) {}
  int next() {
    t.n = 0;
    blocks = 0;
    std::fill(set_blocks, set_blocks + NORM_SETS, 0u);
    int64_t chunks = 0;
    for (; at < n && t.n < MAX_TENSORS; ++at) {
      const pr_grad_tensor &g = tensors[at];
      if (g.numel == 0) continue;
      t.grad[t.n] = g.grad;
      t.numel[t.n] = g.numel;
      t.dtype[t.n] = (unsigned char)g.dtype;
      t.set[t.n] = (unsigned char)g.set;
      chunks += (g.numel + CHUNK - 1) / CHUNK;
      ++t.n;
    }
    // two chunks a workgroup at least, more where that would be too many workgroups
    const int64_t per = std::max<int64_t>((chunks + MAX_BLOCKS - 1) / MAX_BLOCKS, 2);
    for (int k = 0; k < t.n; ++k) {
      const int64_t c = (t.numel[k] + CHUNK - 1) / CHUNK;
      const unsigned b = (unsigned)((c + per - 1) / per);
      t.first_block[k] = blocks;
      blocks += b;
      set_blocks[t.set[k]] += b;
    }
    t.first_block[t.n] = blocks;
    return PR_OK;
  }
};

// Whether no two tensors share memory (scaling them in one launch would race).
int check_apart(const pr_grad_tensor *tensors, int n) {
  struct Span {
    uintptr_t lo, hi;
  };
  Span *s = (Span *)malloc(sizeof(Span) * (size_t)std::max(n, 1));
  if (!s) return PR_ESCRATCH;
  int m = 0;
  for (int i = 0; i < n; ++i) {
    const uintptr_t lo = (uintptr_t)tensors[i].grad;
    if (tensors[i].numel > 0) s[m++] = Span{lo, lo + (uintptr_t)tensors[i].numel * (tensors[i].dtype == PR_F32 ? 4 : 2)};
  }
  std::sort(s, s + m, [](const Span &a, const Span &b) { return a.lo < b.lo; });
  bool apart = true;
  for (int i = 1; i < m; ++i) apart &= s[i - 1].hi <= s[i].lo;
  free(s);
  if (apart) return PR_OK;
  set_error_text("pr_grad_clip: two gradients share memory");
  return PR_EUNSUPPORTED;
}

template <int KIND>
int launch_kind(const pr_grad_tensor *tensors, int n, int n_sets, unsigned joins, double *partials, size_t room,
                NormSets *sets, hipStream_t st) {
  unsigned of_set[NORM_SETS] = {};
  size_t used = 0;
  for (Launches l(tensors, n);;) {
    l.next();
    if (l.t.n == 0) break;
    if (used + l.blocks > room) return PR_ESCRATCH;
    hipLaunchKernelGGL(grad_norm_kernel<KIND>, dim3(l.blocks), dim3(BLOCK), 0, st, l.t, partials + used);
    const int rc = check_launch("pr_grad_norm");
    if (rc != PR_OK) return rc;
    used += l.blocks;
    for (int s = 0; s < n_sets; ++s) of_set[s] += l.set_blocks[s];
  }
  // tensors are ordered by set: a set's partials are consecutive, over launches too
  sets->partials = partials;
  sets->first[0] = 0;
  unsigned most = 0;
  for (int s = 0; s < n_sets; ++s) {
    sets->first[s + 1] = sets->first[s] + of_set[s];
    most = std::max(most, of_set[s]);
  }
  if (most <= joins) return PR_OK;
  if (used + n_sets > room) return PR_ESCRATCH;
  hipLaunchKernelGGL(grad_norm_finish_kernel<KIND>, dim3(n_sets), dim3(BLOCK), 0, st, *sets, partials + used, (float *)nullptr);
  sets->partials = partials + used;
  for (int s = 0; s <= n_sets; ++s) sets->first[s] = s;
  return check_launch("pr_grad_norm");
}

}  // namespace

int check_grad_tensors(const pr_grad_tensor *tensors, int n, int n_sets) {
  if (n < 0 || n_sets < 1 || n_sets > NORM_SETS || (n > 0 && !tensors)) return PR_EINVAL;
  for (int i = 0; i < n; ++i) {
    const pr_grad_tensor &g = tensors[i];
    if (g.numel < 0 || g.numel > (1ll << 38) || (g.numel > 0 && !g.grad) || g.dtype < PR_F32 || g.dtype > PR_BF16) return PR_EINVAL;
    if (((uintptr_t)g.grad & (g.dtype == PR_F32 ? 3 : 1)) != 0) return PR_EINVAL;
    if (g.set < 0 || g.set >= n_sets || (i > 0 && g.set < tensors[i - 1].set)) return PR_EINVAL;
  }
  return PR_OK;
}

size_t grad_norm_scratch(const pr_grad_tensor *tensors, int n) {
  Launches l(tensors, n);
  size_t blocks = NORM_SETS;
  do {
    l.next();
    blocks += l.blocks;
  } while (l.t.n > 0);
  return blocks * sizeof(double);
}

int write_empty_norms(const pr_grad_tensor *tensors, int n, int n_sets, void *scratch, size_t scratch_bytes, float *norms,
                      void *stream) {
  for (int s = 0; s < n_sets; ++s) {
    int64_t elements = 0;
    for (int i = 0; i < n; ++i) elements += tensors[i].set == s ? tensors[i].numel : 0;
    if (elements == 0) return pr_grad_norm(tensors, n, n_sets, PR_NORM_2, scratch, scratch_bytes, norms, stream);
  }
  return PR_OK;
}

int launch_grad_norms(const pr_grad_tensor *tensors, int n, int n_sets, int kind, unsigned joins, void *scratch,
                      size_t scratch_bytes, NormSets *sets, hipStream_t st) {
  double *partials = (double *)scratch;
  const size_t room = scratch_bytes / sizeof(double);
  if (kind == PR_NORM_1) return launch_kind<PR_NORM_1>(tensors, n, n_sets, joins, partials, room, sets, st);
  if (kind == PR_NORM_2) return launch_kind<PR_NORM_2>(tensors, n, n_sets, joins, partials, room, sets, st);
  return launch_kind<PR_NORM_INF>(tensors, n, n_sets, joins, partials, room, sets, st);
}

namespace {
template <int KIND>
int scale_by_norms(const pr_grad_tensor *tensors, int n, const NormSets &sets, const MaxNorms &m, float *norms, hipStream_t st) {
  for (Launches l(tensors, n);;) {
    l.next();
    if (l.t.n == 0) return PR_OK;
    hipLaunchKernelGGL(grad_scale_kernel<KIND>, dim3(l.blocks), dim3(BLOCK), 0, st, l.t, sets, m, norms);
    const int rc = check_launch("pr_grad_clip");
    if (rc != PR_OK) return rc;
  }
}

int check_norm_call(const pr_grad_tensor *tensors, int n, int n_sets, int kind, const void *scratch, size_t scratch_bytes,
                    const float *norms) {
  const int rc = check_grad_tensors(tensors, n, n_sets);
  if (rc != PR_OK) return rc;
  if (kind < PR_NORM_1 || kind > PR_NORM_INF || !norms || !scratch || ((uintptr_t)scratch & 7)) return PR_EINVAL;
  return scratch_bytes < grad_norm_scratch(tensors, n) ? PR_ESCRATCH : PR_OK;
}
}  // namespace
}  // namespace pr

extern "C" int pr_grad_norm_max_sets(void) { return pr::NORM_SETS; }

extern "C" size_t pr_grad_norm_scratch_bytes(const pr_grad_tensor *tensors, int n, int n_sets) {
  return pr::check_grad_tensors(tensors, n, n_sets) == PR_OK ? pr::grad_norm_scratch(tensors, n) : 0;
}

extern "C" int pr_grad_norm(const pr_grad_tensor *tensors, int n, int n_sets, int kind, void *scratch,
                            size_t scratch_bytes, float *norms, void *stream) {
  int rc = pr::check_norm_call(tensors, n, n_sets, kind, scratch, scratch_bytes, norms);
  if (rc != PR_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  pr::NormSets sets;
  rc = pr::launch_grad_norms(tensors, n, n_sets, kind, pr::SCALE_JOINS, scratch, scratch_bytes, &sets, st);
  if (rc != PR_OK) return rc;
  const dim3 grid(n_sets), block(pr::BLOCK);
  double *const none = nullptr;
  if (kind == PR_NORM_2) hipLaunchKernelGGL(pr::grad_norm_finish_kernel<PR_NORM_2>, grid, block, 0, st, sets, none, norms);
  else if (kind == PR_NORM_1) hipLaunchKernelGGL(pr::grad_norm_finish_kernel<PR_NORM_1>, grid, block, 0, st, sets, none, norms);
  else hipLaunchKernelGGL(pr::grad_norm_finish_kernel<PR_NORM_INF>, grid, block, 0, st, sets, none, norms);
  return pr::check_launch("pr_grad_norm");
}

extern "C" int pr_grad_clip(const pr_grad_tensor *tensors, int n, int n_sets, int kind, const double *max_norms,
                            void *scratch, size_t scratch_bytes, float *norms, void *stream) {
  int rc = pr::check_norm_call(tensors, n, n_sets, kind, scratch, scratch_bytes, norms);
  if (rc != PR_OK) return rc;
  if (!max_norms) return PR_EINVAL;
  rc = pr::check_apart(tensors, n);
  if (rc != PR_OK) return rc;
  pr::MaxNorms m{};
  for (int s = 0; s < n_sets; ++s) {
    if (!(max_norms[s] >= 0.0)) return PR_EINVAL;
    m.of[s] = max_norms[s];
  }
  rc = pr::write_empty_norms(tensors, n, n_sets, scratch, scratch_bytes, norms, stream);
  if (rc != PR_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  pr::NormSets sets;
  rc = pr::launch_grad_norms(tensors, n, n_sets, kind, pr::SCALE_JOINS, scratch, scratch_bytes, &sets, st);
  if (rc != PR_OK) return rc;
  if (kind == PR_NORM_1) return pr::scale_by_norms<PR_NORM_1>(tensors, n, sets, m, norms, st);
  if (kind == PR_NORM_2) return pr::scale_by_norms<PR_NORM_2>(tensors, n, sets, m, norms, st);
  return pr::scale_by_norms<PR_NORM_INF>(tensors, n, sets, m, norms, st);
}
