// Global gradient norm and clipping over a list of tensors:
//   norm = sqrt(sum over all entries of (grad_scale g)^2)      out = g grad_scale min(1, max_norm / norm)
// The list travels in the kernel arguments (LIST_MAX tensors per launch), cut into chunks of LIST_CHUNK elements that
// NORM_BLOCKS workgroups take in turn.  Squares are summed in fp64 - no gradient of a finite type overflows or vanishes -
// and every sum has a fixed order, so a norm has the same bits in every run.  Two passes over the data with one
// dependency between them: the second pass' workgroups each add the NORM_BLOCKS partial sums again (8 KiB out of L2)
// instead of waiting for a third launch.
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.h"
#include "kernels.h"

namespace nmtgan {

constexpr int LIST_MAX = 96, LIST_CHUNK = 16384, NORM_BLOCKS = 1024;

struct ListEntry { const void* g; void* out; int64_t n; int first_chunk; int16_t dtype, out_dtype; };
struct ListParams { ListEntry e[LIST_MAX]; int n, n_chunks; };

// four consecutive elements; rows of a list may start at any element, so the vector types promise no more than that
template <typename T> struct Four;
template <> struct Four<float> {
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
  __device__ static __forceinline__ void load(const float* p, float (&x)[4]) {
    const vec v = *reinterpret_cast<const vec*>(p);
    x[0] = v[0]; x[1] = v[1]; x[2] = v[2]; x[3] = v[3];
  }
  __device__ static __forceinline__ void store(float* p, const float (&x)[4]) {
    *reinterpret_cast<vec*>(p) = vec{x[0], x[1], x[2], x[3]};
  }
};
template <typename T> struct Four {
  typedef unsigned vec __attribute__((ext_vector_type(2), aligned(2)));
  __device__ static __forceinline__ void load(const T* p, float (&x)[4]) {
    const vec v = *reinterpret_cast<const vec*>(p);
    Pack16<T>::unpack2(v[0], x[0], x[1]);
    Pack16<T>::unpack2(v[1], x[2], x[3]);
  }
  __device__ static __forceinline__ void store(T* p, const float (&x)[4]) {
    *reinterpret_cast<vec*>(p) = vec{Pack16<T>::pack2(x[0], x[1]), Pack16<T>::pack2(x[2], x[3])};
  }
};

__device__ __forceinline__ int entry_of(const ListParams& p, int chunk) {
  int a = 0, b = p.n - 1;                          // last entry whose first chunk is <= chunk
  while (a < b) {
    const int m = (a + b + 1) / 2;
    if (p.e[m].first_chunk <= chunk) a = m; else b = m - 1;
  }
  return a;
}

__device__ __forceinline__ double block_sum_d(double v, double* red) {
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = (red[0] + red[1]) + (red[2] + red[3]);
  __syncthreads();
  return v;
}

template <typename T>
__device__ __forceinline__ double square_sum(const T* g, int n) {
  double s = 0.0;
  const int n4 = n / 4;
  for (int i = threadIdx.x; i < n4; i += 256) {
    float x[4];
    Four<T>::load(g + 4 * i, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fma((double)x[e], (double)x[e], s);
  }
  for (int i = 4 * n4 + threadIdx.x; i < n; i += 256) {
    const double x = OpTraits<T>::load(g + i);
    s = fma(x, x, s);
  }
  return s;
}

__global__ __launch_bounds__(256) void norm_kernel(ListParams p, double* part) {
  __shared__ double red[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < p.n_chunks; c += NORM_BLOCKS) {
    const ListEntry& e = p.e[entry_of(p, c)];
    const int64_t off = (int64_t)(c - e.first_chunk) * LIST_CHUNK;
    const int n = (int)min((int64_t)LIST_CHUNK, e.n - off);
    if (e.dtype == NMTGAN_F32) s += square_sum((const float*)e.g + off, n);
    else if (e.dtype == NMTGAN_F16) s += square_sum((const f16_t*)e.g + off, n);
    else s += square_sum((const bf16_t*)e.g + off, n);
  }
  s = block_sum_d(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double total_norm(const double* part, int n, float grad_scale, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s += part[i];
  return sqrt(block_sum_d(s, red)) * fabs((double)grad_scale);
}

__global__ __launch_bounds__(256) void norm_finish_kernel(const double* part, int n, float grad_scale, float* norm) {
  __shared__ double red[4];
  const double t = total_norm(part, n, grad_scale, red);
  if (threadIdx.x == 0) norm[0] = (float)t;
}

template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T* g, O* out, int n, float f) {
  const int n4 = n / 4;
  for (int i = threadIdx.x; i < n4; i += 256) {
    float x[4];
    Four<T>::load(g + 4 * i, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= f;
    Four<O>::store(out + 4 * i, x);
  }
  for (int i = 4 * n4 + threadIdx.x; i < n; i += 256) OpTraits<O>::store(out + i, OpTraits<T>::load(g + i) * f);
}

__global__ __launch_bounds__(256) void clip_kernel(ListParams p, const double* part, int n_part, float grad_scale,
                                                   float max_norm, float* norm) {
  __shared__ double red[4];
  const double t = total_norm(part, n_part, grad_scale, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)t;
  // a norm that is no finite number makes every output NaN, as tf.clip_by_global_norm does: the step is seen to be lost
  const float f = !(t < INFINITY) ? NAN : (t > (double)max_norm ? (float)((double)max_norm / t * (double)grad_scale) : grad_scale);
  for (int c = blockIdx.x; c < p.n_chunks; c += gridDim.x) {
    const ListEntry& e = p.e[entry_of(p, c)];
    if (f == 1.f && e.out == e.g) continue;          // nothing to change in place
    const int64_t off = (int64_t)(c - e.first_chunk) * LIST_CHUNK;
    const int n = (int)min((int64_t)LIST_CHUNK, e.n - off);
    if (e.dtype == NMTGAN_F32) scale_chunk((const float*)e.g + off, (float*)e.out + off, n, f);
    else if (e.dtype == NMTGAN_F16) {
      if (e.out_dtype == NMTGAN_F32) scale_chunk((const f16_t*)e.g + off, (float*)e.out + off, n, f);
      else scale_chunk((const f16_t*)e.g + off, (f16_t*)e.out + off, n, f);
    } else {
      if (e.out_dtype == NMTGAN_F32) scale_chunk((const bf16_t*)e.g + off, (float*)e.out + off, n, f);
      else scale_chunk((const bf16_t*)e.g + off, (bf16_t*)e.out + off, n, f);
    }
  }
}

static int check_list(const nmtgan_grad_ref* t, int n, bool clip, const char* what) {
  NMTGAN_REQUIRE(n >= 0 && (n == 0 || t), "%s: null list", what);
  struct Range { uintptr_t a, b; int tensor; };
  std::vector<Range> written, read;
  for (int i = 0; i < n; ++i) {
    NMTGAN_REQUIRE(t[i].n >= 0 && valid_op_dtype(t[i].dtype), "%s: tensor %d: bad size or dtype", what, i);
    NMTGAN_REQUIRE(t[i].n < (1LL << 40), "%s: tensor %d: too large", what, i);
    if (t[i].n == 0) continue;
    const int es = dtype_size(t[i].dtype);
    NMTGAN_REQUIRE(t[i].g && (uintptr_t)t[i].g % es == 0, "%s: tensor %d: null or misaligned", what, i);
    if (!clip) continue;
    const int oes = dtype_size(t[i].out_dtype);
    NMTGAN_REQUIRE(t[i].out && (uintptr_t)t[i].out % oes == 0, "%s: tensor %d: null or misaligned output", what, i);
    NMTGAN_REQUIRE(t[i].out_dtype == t[i].dtype || t[i].out_dtype == NMTGAN_F32,
                   "%s: tensor %d: the output has the gradient's type or is fp32", what, i);
    NMTGAN_REQUIRE(t[i].out != t[i].g || es == oes, "%s: tensor %d: in place needs equal types", what, i);
    written.push_back({(uintptr_t)t[i].out, (uintptr_t)t[i].out + (uintptr_t)(t[i].n * oes), i});
    if (t[i].out != t[i].g) read.push_back({(uintptr_t)t[i].g, (uintptr_t)t[i].g + (uintptr_t)(t[i].n * es), i});
  }
  // a place that is written twice, or read by one workgroup and written by another, has no defined result
  auto before = [](const Range& x, const Range& y) { return x.a < y.a; };
  std::sort(written.begin(), written.end(), before);
  for (size_t i = 1; i < written.size(); ++i)
    NMTGAN_REQUIRE(written[i].a >= written[i - 1].b, "%s: outputs of tensors %d and %d overlap", what, written[i - 1].tensor,
                   written[i].tensor);
  for (const Range& r : read) {
    auto it = std::upper_bound(written.begin(), written.end(), r, before);
    const bool hit = (it != written.end() && it->a < r.b) || (it != written.begin() && (it - 1)->b > r.a);
    NMTGAN_REQUIRE(!hit, "%s: tensor %d overlaps an output", what, r.tensor);
  }
  return 0;
}

// launches fn(list part, index) for every run of at most LIST_MAX non-empty tensors whose chunks fit an int
template <typename F>
static int for_parts(const nmtgan_grad_ref* t, int n, F fn) {
  ListParams p{};
  int k = 0;
  auto flush = [&]() -> int {
    if (p.n == 0) return 0;
    const int rc = fn(p, k++);
    p.n = 0;
    p.n_chunks = 0;
    return rc;
  };
  for (int i = 0; i < n; ++i) {
    if (t[i].n == 0) continue;
    const int64_t c = (t[i].n + LIST_CHUNK - 1) / LIST_CHUNK;
    if (p.n == LIST_MAX || p.n_chunks + c > (1LL << 30)) NMTGAN_TRY(flush());
    p.e[p.n++] = ListEntry{t[i].g, t[i].out, t[i].n, p.n_chunks, (int16_t)t[i].dtype, (int16_t)t[i].out_dtype};
    p.n_chunks += (int)c;
  }
  return flush();
}
static int list_parts(const nmtgan_grad_ref* t, int n) {
  int k = 0;
  (void)for_parts(t, n, [&](const ListParams&, int) { ++k; return 0; });
  return k;
}

size_t global_norm_workspace(int n_tensors) {
  return (size_t)((std::max(n_tensors, 1) + LIST_MAX - 1) / LIST_MAX + 2) * NORM_BLOCKS * sizeof(double);
}
static int sum_squares(const nmtgan_grad_ref* t, int n, void* ws, size_t ws_bytes, int* n_part, const char* what, hipStream_t st) {
  const size_t need = (size_t)std::max(1, list_parts(t, n)) * NORM_BLOCKS * sizeof(double);
  NMTGAN_REQUIRE(ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0, "%s: workspace of %zu bytes needed, %zu given", what, need,
                 ws_bytes);
  *n_part = 0;
  return for_parts(t, n, [&](const ListParams& p, int k) -> int {
    hipLaunchKernelGGL(norm_kernel, dim3(NORM_BLOCKS), dim3(256), 0, st, p, (double*)ws + (int64_t)k * NORM_BLOCKS);
    NMTGAN_CHECK_LAUNCH("global_norm");
    *n_part = (k + 1) * NORM_BLOCKS;
    return 0;
  });
}
int launch_global_norm(const nmtgan_grad_ref* t, int n, float grad_scale, float* norm, void* ws, size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  NMTGAN_TRY(check_list(t, n, false, "global_norm"));
  NMTGAN_REQUIRE(norm && isfinite(grad_scale), "global_norm: null norm or bad scale");
  int n_part = 0;
  NMTGAN_TRY(sum_squares(t, n, ws, ws_bytes, &n_part, "global_norm", st));
  hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(256), 0, st, (const double*)ws, n_part, grad_scale, norm);
  NMTGAN_CHECK_LAUNCH("global_norm_finish");
  return 0;
}
int launch_clip_global_norm(const nmtgan_grad_ref* t, int n, float max_norm, float grad_scale, float* norm, void* ws,
                            size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  NMTGAN_TRY(check_list(t, n, true, "clip_global_norm"));
  NMTGAN_REQUIRE(norm && isfinite(grad_scale), "clip_global_norm: null norm or bad scale");
  NMTGAN_REQUIRE(max_norm > 0.f && isfinite(max_norm), "clip_global_norm: max_norm must be positive and finite");
  int n_part = 0;
  NMTGAN_TRY(sum_squares(t, n, ws, ws_bytes, &n_part, "clip_global_norm", st));
  if (n_part == 0) {
    hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(256), 0, st, (const double*)ws, 0, grad_scale, norm);
    NMTGAN_CHECK_LAUNCH("clip_global_norm");
    return 0;
  }
  return for_parts(t, n, [&](const ListParams& p, int k) -> int {
    const int grid = std::min(p.n_chunks, 2 * NORM_BLOCKS);
    hipLaunchKernelGGL(clip_kernel, dim3(grid), dim3(256), 0, st, p, (const double*)ws, n_part, grad_scale, max_norm,
                       k == 0 ? norm : nullptr);
    NMTGAN_CHECK_LAUNCH("clip_global_norm");
    return 0;
  });
}

}  // namespace nmtgan
