// Global gradient norm and clipping over a list of tensors:
//   norm = sqrt(sum over all entries of (grad_scale g)^2)      out = g grad_scale min(1, max_norm / norm)
// The list travels in the kernel arguments (LIST_MAX tensors per launch), cut into chunks of LIST_CHUNK elements that
// up to NORM_BLOCKS workgroups take in turn.  Squares are summed in fp64 - no gradient of a finite type overflows or vanishes -
// and every sum has a fixed order, so a norm has the same bits in every run.  Two passes over the data with one
// dependency between them: the second pass' workgroups each add the partial sums again (out of L2, up to 8 KiB for every
// LIST_MAX tensors: 16 KiB below) instead of waiting for another launch.  Bound by memory: the 195 tensors and 93 million entries of a six-block generator
// with its tables (16 bits, two launches of each kernel): norm 52 us, clip into an fp32 buffer 102 us = 5.5 TB/s.  1600 tensors of
// 262144 elements, ten launches of each: norm 194 us, both 799 us, 4.2 TB/s.
#include <math.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "common.h"
#include "kernels.h"

namespace nmtgan {

constexpr int LIST_MAX = 160, LIST_CHUNK = 16384, NORM_BLOCKS = 1024;

// a tensor takes chunks [first_chunk, first_chunk of the next entry); tail = elements of its last one and the two dtypes
struct ListEntry { const void* g; void* out; int first_chunk; unsigned tail; };
struct ListParams { ListEntry e[LIST_MAX]; int n, n_chunks; };
static_assert(sizeof(ListParams) + 64 <= 4096, "the list travels as kernel arguments (4 KB)");
static inline unsigned pack_tail(int n, int dtype, int out_dtype) {
  return (unsigned)n | (unsigned)dtype << 20 | (unsigned)out_dtype << 24;
}

// 16 bytes / four elements at any element of a tensor: the vector types promise no more than an element's alignment
typedef unsigned u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename T> struct Any {
  using vec4 = std::conditional_t<sizeof(T) == 4, u32x4_at4, u32x4_at2>;
  using vec2 = u32x2_at2;
  static constexpr int E = 16 / (int)sizeof(T);
  __device__ static __forceinline__ uint4 load16(const T* p) {
    const vec4 v = *reinterpret_cast<const vec4*>(p);
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  __device__ static __forceinline__ void unpack(const uint4& r, float (&x)[E]) {
    if constexpr (sizeof(T) == 2) {
      unpack8<T>(r, x);
    } else {
      x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    }
  }
  __device__ static __forceinline__ void load4(const T* p, float (&x)[4]) {
    if constexpr (sizeof(T) == 2) {
      const vec2 v = *reinterpret_cast<const vec2*>(p);
      Pack16<T>::unpack2(v[0], x[0], x[1]);
      Pack16<T>::unpack2(v[1], x[2], x[3]);
    } else {
      const vec4 v = *reinterpret_cast<const vec4*>(p);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
    }
  }
  __device__ static __forceinline__ void store4(T* p, const float (&x)[4]) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<vec2*>(p) = vec2{Pack16<T>::pack2(x[0], x[1]), Pack16<T>::pack2(x[2], x[3])};
    } else {
      *reinterpret_cast<vec4*>(p) =
          vec4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    }
  }
};

// entry of a chunk, the chunk's first element inside the tensor and its length
__device__ __forceinline__ const ListEntry& chunk_of(const ListParams& p, int chunk, int64_t& off, int& n) {
  // last entry whose first chunk is <= chunk: all entries at once, a search by halves waits for a load at every step
  int a = -1;
#pragma unroll
  for (int u = 0; u < (LIST_MAX + 63) / 64; ++u) {
    const int i = 64 * u + (threadIdx.x & 63);
    a += __popcll(__ballot(i < p.n && p.e[min(i, LIST_MAX - 1)].first_chunk <= chunk));
  }
  const ListEntry& e = p.e[a];
  off = (int64_t)(chunk - e.first_chunk) * LIST_CHUNK;
  n = chunk + 1 == (a + 1 < p.n ? p.e[a + 1].first_chunk : p.n_chunks) ? (int)(e.tail & 0xfffff) : LIST_CHUNK;
  return e;
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
  constexpr int E = Any<T>::E, U = 8;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
  int i = 0;
  for (; i + 256 * E * U <= n; i += 256 * E * U) {           // eight loads in flight
    uint4 r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = Any<T>::load16(g + i + (u * 256 + (int)threadIdx.x) * E);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[E];
      Any<T>::unpack(r[u], x);
#pragma unroll
      for (int e = 0; e < E; ++e) s[e & 3] = fma((double)x[e], (double)x[e], s[e & 3]);
    }
  }
  for (i += threadIdx.x * E; i < n; i += 256 * E) {
    if (i + E <= n) {
      float x[E];
      Any<T>::unpack(Any<T>::load16(g + i), x);
#pragma unroll
      for (int e = 0; e < E; ++e) s[e & 3] = fma((double)x[e], (double)x[e], s[e & 3]);
    } else {
      for (int k = i; k < n; ++k) {
        const double x = OpTraits<T>::load(g + k);
        s[0] = fma(x, x, s[0]);
      }
    }
  }
  return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(256) void norm_kernel(ListParams p, double* part) {
  __shared__ double red[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < p.n_chunks; c += gridDim.x) {
    int64_t off;
    int n;
    const ListEntry& e = chunk_of(p, c, off, n);
    const int dtype = e.tail >> 20 & 15;
    if (dtype == NMTGAN_F32) s += square_sum((const float*)e.g + off, n);
    else if (dtype == NMTGAN_F16) s += square_sum((const f16_t*)e.g + off, n);
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
__device__ __forceinline__ void scale_chunk(const T* g, O* out, int n, float pre, float f) {
  constexpr int U = 8;
  int i = 0;
  for (; i + 1024 * U <= n; i += 1024 * U) {
    float x[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) Any<T>::load4(g + i + (u * 256 + (int)threadIdx.x) * 4, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[u][e] = x[u][e] * pre * f;
      Any<O>::store4(out + i + (u * 256 + (int)threadIdx.x) * 4, x[u]);
    }
  }
  for (i += threadIdx.x * 4; i < n; i += 1024) {
    if (i + 4 <= n) {
      float x[4];
      Any<T>::load4(g + i, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = x[e] * pre * f;
      Any<O>::store4(out + i, x);
    } else {
      for (int k = i; k < n; ++k) OpTraits<O>::store(out + k, OpTraits<T>::load(g + k) * pre * f);
    }
  }
}

__global__ __launch_bounds__(256) void clip_kernel(ListParams p, const double* part, int n_part, float grad_scale,
                                                   float max_norm, float* norm) {
  __shared__ double red[4];
  const double t = total_norm(part, n_part, grad_scale, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)t;
  // a norm that is no finite number makes every output NaN: the step is seen to be lost
  const double all = !(t < INFINITY) ? NAN : (t > (double)max_norm ? (double)max_norm / t * (double)grad_scale : (double)grad_scale);
  // a factor below fp32's normal range, of a norm above 8e37 max_norm, goes in two: the values it makes are not that small
  const bool tiny = fabs(all) < 0x1p-126;
  const float pre = tiny ? 0x1p-126f : 1.f, f = (float)(tiny ? all * 0x1p126 : all);
  for (int c = blockIdx.x; c < p.n_chunks; c += gridDim.x) {
    int64_t off;
    int n;
    const ListEntry& e = chunk_of(p, c, off, n);
    if (f == 1.f && !tiny && e.out == e.g) continue;          // nothing to change in place
    const int dtype = e.tail >> 20 & 15, out_dtype = e.tail >> 24 & 15;
    if (dtype == NMTGAN_F32) scale_chunk((const float*)e.g + off, (float*)e.out + off, n, pre, f);
    else if (dtype == NMTGAN_F16) {
      if (out_dtype == NMTGAN_F32) scale_chunk((const f16_t*)e.g + off, (float*)e.out + off, n, pre, f);
      else scale_chunk((const f16_t*)e.g + off, (f16_t*)e.out + off, n, pre, f);
    } else {
      if (out_dtype == NMTGAN_F32) scale_chunk((const bf16_t*)e.g + off, (float*)e.out + off, n, pre, f);
      else scale_chunk((const bf16_t*)e.g + off, (bf16_t*)e.out + off, n, pre, f);
    }
  }
}

static int check_list(const nmtgan_grad_ref* t, int n, bool clip, const char* what) {
  NMTGAN_REQUIRE(n >= 0 && (n == 0 || t), "%s: null list", what);
  struct Range { uintptr_t a, b; int tensor; };
  std::vector<Range> written, read;
  written.reserve(clip ? n : 0);
  read.reserve(clip ? n : 0);
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
    p.e[p.n++] = ListEntry{t[i].g, t[i].out, p.n_chunks, pack_tail((int)(t[i].n - (c - 1) * LIST_CHUNK), t[i].dtype, t[i].out_dtype)};
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
  return for_parts(t, n, [&](const ListParams& p, int) -> int {
    const int grid = std::min(p.n_chunks, NORM_BLOCKS);
    hipLaunchKernelGGL(norm_kernel, dim3(grid), dim3(256), 0, st, p, (double*)ws + *n_part);
    NMTGAN_CHECK_LAUNCH("global_norm");
    *n_part += grid;
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
