// Span attention: query row i attends to the keys lo[i] <= j < hi[i] of one packed key buffer.  Causal, document, prefix
// and padding masks of a packed (or padded) batch are all spans, so one kernel family serves teacher-forced training on
// packed sentences, prompts, and single tokens over a long cache.
//
//   r = scale q_i . k_j          t = tanh(r / cap), s = cap t   (s = r without a cap)
//   s -= slope_h |pos_i - j|     p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij)       out_i = sum_j p_ij v_j
//   dp = dout_i . v_j   delta_i = dout_i . out_i   dr = p (dp - delta_i) (1 - t^2) scale
//   dq_i = sum_j dr k_j    dk_j = sum_i dr q_i    dv_j = sum_i p dout_i   (sums over the heads that share a key head too)
//
// The row functions below do one row by one wave with plain fp32 arithmetic; they touch visible (row, key) pairs only,
// so whatever sits in rows outside the spans (NaN and infinities included) stays outside the result.
#include <math.h>

#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace nmtgan {

constexpr int SPAN_MAX_DH = 128;
constexpr float LOG2E = 1.44269504088896341f;

struct SpanParams {
  const void* q; const void* k; const void* v;
  int64_t ldq, ldk, ldv, ldo;
  const int32_t* lo; const int32_t* hi; const int32_t* pos;
  const float* slopes;
  void* out; float* lse;
  int M, N, heads, kv_heads, dh;
  float scale, cap;
  // gradients
  const void* dout; int64_t ld_do;
  void* dq; void* dk; void* dv;
  int64_t ld_dq, ld_dk, ld_dv;
  float* delta;                                  // [M][heads]
  int2* hull;                                    // [ceil(M / 64)] keys seen by any row of the block
};

__device__ __forceinline__ float span_exp(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// span of row i, cut to the key buffer; an empty one is (0, 0)
__device__ __forceinline__ int2 span_of(const SpanParams& p, int i) {
  const int a = max(p.lo[i], 0), b = min(p.hi[i], p.N);
  return b > a ? make_int2(a, b) : make_int2(0, 0);
}
__device__ __forceinline__ int pos_of(const SpanParams& p, int i) { return p.pos ? p.pos[i] : p.hi[i] - 1; }

// score of a raw product and the factor d(score)/d(product)
__device__ __forceinline__ float span_score(const SpanParams& p, float dot, float slope, int pos, int j, float& turn) {
  float r = dot * p.scale;
  turn = p.scale;
  if (p.cap > 0.f) {
    const float t = tanhf(r / p.cap);
    r = p.cap * t;
    turn = (1.f - t * t) * p.scale;
  }
  if (p.slopes) r -= slope * fabsf((float)(pos - j));
  return r;
}

// dot product of dh elements at `row` with the fp32 vector x (LDS, the same address in every lane)
template <typename T>
__device__ __forceinline__ float dot_row(const T* row, const float* x, int dh) {
  float s = 0.f;
  for (int c = 0; c < dh; c += 8) {
    float a[8];
    VecIO<T, 8>::load(row + c, a);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(a[e], x[c + e], s);
  }
  return s;
}
template <typename T>
__device__ __forceinline__ void stage_row(const T* row, float* x, int dh, int lane) {
  for (int c = lane; c < dh; c += 64) x[c] = OpTraits<T>::load(row + c);
}

template <typename T>
__device__ void span_fwd_row(const SpanParams& p, int i, int h, float* x, int lane) {
  const int dh = p.dh, kvh = h / (p.heads / p.kv_heads);
  const T* K = (const T*)p.k + kvh * dh;
  const T* V = (const T*)p.v + kvh * dh;
  stage_row((const T*)p.q + i * p.ldq + h * dh, x, dh, lane);
  __builtin_amdgcn_wave_barrier();
  const int2 sp = span_of(p, i);
  const int pos = pos_of(p, i);
  const float slope = p.slopes ? p.slopes[h] : 0.f;
  float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
  for (int j0 = sp.x; j0 < sp.y; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY, turn;
    if (j < sp.y) s = span_score(p, dot_row(K + j * p.ldk, x, dh), slope, pos, j, turn);
    const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float pe = j < sp.y ? span_exp(s - mu) : 0.f, f = span_exp(m - mu);
    l = l * f + wave_sum(pe);
    acc[0] *= f;
    acc[1] *= f;
    m = mn;
    const int n = min(64, sp.y - j0);
    for (int t = 0; t < n; ++t) {
      const float pt = __shfl(pe, t, 64);
      const T* row = V + (j0 + t) * p.ldv;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < dh) acc[u] = fmaf(pt, OpTraits<T>::load(row + lane + 64 * u), acc[u]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;               // NaN stays NaN
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 64 * u < dh) OpTraits<T>::store((T*)p.out + i * p.ldo + h * dh + lane + 64 * u, l == 0.f ? 0.f : acc[u] * inv);
  if (p.lse && lane == 0) p.lse[(int64_t)i * p.heads + h] = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + logf(l);
  __builtin_amdgcn_wave_barrier();
}

// p_ij and dr_ij of lane's pair; x = q row, y = dout row
template <typename T>
__device__ __forceinline__ void span_pair(const SpanParams& p, const T* krow, const T* vrow, const float* x, const float* y,
                                          float lse, float delta, float slope, int pos, int j, float& pe, float& dr) {
  float turn;
  const float s = span_score(p, dot_row(krow, x, p.dh), slope, pos, j, turn);
  pe = lse == -INFINITY ? 0.f : span_exp(s - lse);
  dr = pe * (dot_row(vrow, y, p.dh) - delta) * turn;
}

template <typename T>
__device__ void span_dq_row(const SpanParams& p, int i, int h, float* x, float* y, int lane) {
  const int dh = p.dh, kvh = h / (p.heads / p.kv_heads);
  const T* K = (const T*)p.k + kvh * dh;
  const T* V = (const T*)p.v + kvh * dh;
  stage_row((const T*)p.q + i * p.ldq + h * dh, x, dh, lane);
  stage_row((const T*)p.dout + i * p.ld_do + h * dh, y, dh, lane);
  __builtin_amdgcn_wave_barrier();
  const int2 sp = span_of(p, i);
  const int pos = pos_of(p, i);
  const float slope = p.slopes ? p.slopes[h] : 0.f;
  const float lse = p.lse[(int64_t)i * p.heads + h], delta = p.delta[(int64_t)i * p.heads + h];
  float acc[2] = {0.f, 0.f};
  for (int j0 = sp.x; j0 < sp.y; j0 += 64) {
    const int j = j0 + lane;
    float pe = 0.f, dr = 0.f;
    if (j < sp.y) span_pair(p, K + j * p.ldk, V + j * p.ldv, x, y, lse, delta, slope, pos, j, pe, dr);
    const int n = min(64, sp.y - j0);
    for (int t = 0; t < n; ++t) {
      const float d = __shfl(dr, t, 64);
      const T* row = K + (j0 + t) * p.ldk;
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < dh) acc[u] = fmaf(d, OpTraits<T>::load(row + lane + 64 * u), acc[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 64 * u < dh) OpTraits<T>::store((T*)p.dq + i * p.ld_dq + h * dh + lane + 64 * u, acc[u]);
  __builtin_amdgcn_wave_barrier();
}

// key j of key head kvh: x = k row, y = v row; walks the query rows that see it, head by head of the group
template <typename T>
__device__ void span_dkv_key(const SpanParams& p, int j, int kvh, float* x, float* y, int lane) {
  const int dh = p.dh, g = p.heads / p.kv_heads;
  stage_row((const T*)p.k + j * p.ldk + kvh * dh, x, dh, lane);
  stage_row((const T*)p.v + j * p.ldv + kvh * dh, y, dh, lane);
  __builtin_amdgcn_wave_barrier();
  float ak[2] = {0.f, 0.f}, av[2] = {0.f, 0.f};
  const int nb = (p.M + 63) / 64;
  for (int b = 0; b < nb; ++b) {
    const int2 hl = p.hull[b];
    if (j < hl.x || j >= hl.y) continue;
    const int i = b * 64 + lane;
    int2 sp = make_int2(0, 0);
    int pos = 0;
    if (i < p.M) { sp = span_of(p, i); pos = pos_of(p, i); }
    const bool on = j >= sp.x && j < sp.y;
    const unsigned long long mask = __ballot(on);
    if (mask == 0) continue;
    for (int h = kvh * g; h < (kvh + 1) * g; ++h) {
      const T* Q = (const T*)p.q + h * dh;
      const T* D = (const T*)p.dout + h * dh;
      float pe = 0.f, dr = 0.f;
      if (on)
        span_pair(p, Q + i * p.ldq, D + i * p.ld_do, x, y, p.lse[(int64_t)i * p.heads + h],
                  p.delta[(int64_t)i * p.heads + h], p.slopes ? p.slopes[h] : 0.f, pos, j, pe, dr);
      for (unsigned long long left = mask; left; left &= left - 1) {
        const int t = __builtin_ctzll(left);
        const float pt = __shfl(pe, t, 64), dt = __shfl(dr, t, 64);
        const int64_t r = b * 64 + t;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (lane + 64 * u < dh) {
            av[u] = fmaf(pt, OpTraits<T>::load(D + r * p.ld_do + lane + 64 * u), av[u]);
            ak[u] = fmaf(dt, OpTraits<T>::load(Q + r * p.ldq + lane + 64 * u), ak[u]);
          }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 64 * u < dh) {
      OpTraits<T>::store((T*)p.dk + j * p.ld_dk + kvh * dh + lane + 64 * u, ak[u]);
      OpTraits<T>::store((T*)p.dv + j * p.ld_dv + kvh * dh + lane + 64 * u, av[u]);
    }
  __builtin_amdgcn_wave_barrier();
}

// ------------------------------------------------------------------------------------------ one wave per row
template <typename T>
__global__ __launch_bounds__(256) void span_fwd_rows_kernel(SpanParams p) {
  __shared__ float xs[4][SPAN_MAX_DH];
  const int w = threadIdx.x >> 6, i = blockIdx.x * 4 + w;
  if (i < p.M) span_fwd_row<T>(p, i, blockIdx.y, xs[w], threadIdx.x & 63);
}
template <typename T>
__global__ __launch_bounds__(256) void span_dq_rows_kernel(SpanParams p) {
  __shared__ float xs[4][2][SPAN_MAX_DH];
  const int w = threadIdx.x >> 6, i = blockIdx.x * 4 + w;
  if (i < p.M) span_dq_row<T>(p, i, blockIdx.y, xs[w][0], xs[w][1], threadIdx.x & 63);
}
template <typename T>
__global__ __launch_bounds__(256) void span_dkv_keys_kernel(SpanParams p) {
  __shared__ float xs[4][2][SPAN_MAX_DH];
  const int w = threadIdx.x >> 6, j = blockIdx.x * 4 + w;
  if (j < p.N) span_dkv_key<T>(p, j, blockIdx.y, xs[w][0], xs[w][1], threadIdx.x & 63);
}

// What the gradient kernels need per row and per 64 rows: delta_i = dout_i . out_i of every head (0 for rows that see
// nothing, whatever their dout holds) and the hull of the spans.  One workgroup per 64 rows; a row's head products are
// summed by 8 lanes.
template <typename T>
__global__ __launch_bounds__(256) void span_prep_kernel(SpanParams p) {
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (w == 0) {
    const int i = b * 64 + lane;
    int2 sp = make_int2(0, 0);
    if (i < p.M) sp = span_of(p, i);
    int a = sp.y > sp.x ? sp.x : 0x7fffffff, e = sp.y;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) { a = min(a, __shfl_xor(a, o, 64)); e = max(e, __shfl_xor(e, o, 64)); }
    if (lane == 0) p.hull[b] = make_int2(a, e);
  }
  const int n = min(64, p.M - b * 64) * p.heads, c8 = p.dh / 8;
  for (int t = threadIdx.x >> 3; t < n; t += 32) {
    const int64_t i = b * 64 + t / p.heads;
    const int h = t % p.heads;
    const T* o = (const T*)p.out + i * p.ldo + h * p.dh;
    const T* d = (const T*)p.dout + i * p.ld_do + h * p.dh;
    float s = 0.f;
    for (int c = threadIdx.x & 7; c < c8; c += 8) {
      float x[8], y[8];
      VecIO<T, 8>::load(o + 8 * c, x);
      VecIO<T, 8>::load(d + 8 * c, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
    }
    s = dpp_add<0xB1>(s);
    s = dpp_add<0x4E>(s);
    s = dpp_add<0x141>(s);
    if ((threadIdx.x & 7) == 0) {
      const int2 sp = span_of(p, (int)i);
      p.delta[i * p.heads + h] = sp.y > sp.x ? s : 0.f;
    }
  }
}

// ------------------------------------------------------------------------------------------ single tokens
// One query row per workgroup and key head, `splits` workgroups along the span; every wave takes every fourth block of
// keys.  part[row][head][split] = (acc[dh], m, l), joined in split order by span_join_kernel.
template <typename T>
__global__ __launch_bounds__(256) void span_step_kernel(SpanParams p, int splits, float* part) {
  __shared__ float xs[4][SPAN_MAX_DH];
  __shared__ float ms[4], ls[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int i = blockIdx.x / splits, z = blockIdx.x % splits, h = blockIdx.y, dh = p.dh;
  const int kvh = h / (p.heads / p.kv_heads);
  const int2 sp = span_of(p, i);
  const int pos = pos_of(p, i), len = sp.y - sp.x;
  const int j0 = sp.x + (int)((int64_t)len * z / splits), j1 = sp.x + (int)((int64_t)len * (z + 1) / splits);
  const float slope = p.slopes ? p.slopes[h] : 0.f;
  const T* K = (const T*)p.k + kvh * dh;
  const T* V = (const T*)p.v + kvh * dh;
  stage_row((const T*)p.q + i * p.ldq + h * dh, xs[w], dh, lane);
  __builtin_amdgcn_wave_barrier();
  float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
  for (int b = j0 + 64 * w; b < j1; b += 256) {
    const int j = b + lane;
    float s = -INFINITY, turn;
    if (j < j1) s = span_score(p, dot_row(K + j * p.ldk, xs[w], dh), slope, pos, j, turn);
    const float mn = fmaxf(m, wave_max(s)), mu = mn == -INFINITY ? 0.f : mn;
    const float pe = j < j1 ? span_exp(s - mu) : 0.f, f = span_exp(m - mu);
    l = l * f + wave_sum(pe);
    m = mn;
    acc[0] *= f;
    acc[1] *= f;
    const int n = min(64, j1 - b);
    for (int t = 0; t < n; ++t) {
      const float pt = __shfl(pe, t, 64);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (lane + 64 * u < dh) acc[u] = fmaf(pt, OpTraits<T>::load(V + (b + t) * p.ldv + lane + 64 * u), acc[u]);
    }
  }
  __syncthreads();
  if (lane == 0) { ms[w] = m; ls[w] = l; }
  __syncthreads();
  const float mt = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), mu = mt == -INFINITY ? 0.f : mt;
  const float f = span_exp(m - mu);
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 64 * u < dh) xs[w][lane + 64 * u] = acc[u] * f;
  __syncthreads();
  float* o = part + (((int64_t)i * p.heads + h) * splits + z) * (dh + 2);
  for (int c = threadIdx.x; c < dh; c += 256) o[c] = (xs[0][c] + xs[1][c]) + (xs[2][c] + xs[3][c]);
  if (threadIdx.x == 0) {
    float lt = 0.f;
    for (int k = 0; k < 4; ++k) lt += ls[k] * span_exp(ms[k] - mu);
    o[dh] = mu;
    o[dh + 1] = lt;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void span_join_kernel(SpanParams p, int splits, const float* part) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= (int64_t)p.M * p.heads) return;
  const int i = (int)(t / p.heads), h = (int)(t % p.heads), dh = p.dh;
  const float* o = part + t * splits * (dh + 2);
  float m = -INFINITY;
  for (int z = 0; z < splits; ++z)
    if (o[z * (dh + 2) + dh + 1] != 0.f) m = fmaxf(m, o[z * (dh + 2) + dh]);
  const float mu = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc[2] = {0.f, 0.f};
  for (int z = 0; z < splits; ++z) {
    const float* q = o + z * (dh + 2);
    if (q[dh + 1] == 0.f) continue;
    const float f = span_exp(q[dh] - mu);
    l += q[dh + 1] * f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (lane + 64 * u < dh) acc[u] += q[lane + 64 * u] * f;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (lane + 64 * u < dh)
      OpTraits<T>::store((T*)p.out + i * p.ldo + h * dh + lane + 64 * u, l == 0.f ? 0.f : acc[u] / l);
  if (p.lse && lane == 0) p.lse[t] = l == 0.f ? -INFINITY : mu + logf(l);
}

// ------------------------------------------------------------------------------------------ host
static bool rows_ok(const void* ptr, int64_t ld, int64_t width, int es) {
  return (uintptr_t)ptr % 16 == 0 && ld >= width && ld * es % 16 == 0;
}
static int fill_span(const nmtgan_span_args* a, SpanParams& p, const char* what) {
  NMTGAN_REQUIRE(a != nullptr, "%s: null args", what);
  NMTGAN_REQUIRE(valid_op_dtype(a->dtype), "%s: bad dtype %d", what, a->dtype);
  NMTGAN_REQUIRE(a->M >= 0 && a->N >= 0, "%s: bad shape M=%d N=%d", what, a->M, a->N);
  NMTGAN_REQUIRE(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->heads <= 4096,
                 "%s: heads=%d must be a multiple of kv_heads=%d, at most 4096", what, a->heads, a->kv_heads);
  NMTGAN_REQUIRE(a->dh > 0 && a->dh % 8 == 0 && a->dh <= SPAN_MAX_DH, "%s: head width %d must be a multiple of 8, at most %d",
                 what, a->dh, SPAN_MAX_DH);
  NMTGAN_REQUIRE(isfinite(a->scale) && isfinite(a->cap) && a->cap >= 0.f, "%s: scale and cap must be finite, cap >= 0", what);
  const int es = dtype_size(a->dtype);
  if (a->M > 0) {
    NMTGAN_REQUIRE(a->q && a->lo && a->hi && a->out, "%s: null pointer", what);
    NMTGAN_REQUIRE(rows_ok(a->q, a->ldq, (int64_t)a->heads * a->dh, es) && rows_ok(a->out, a->ldo, (int64_t)a->heads * a->dh, es),
                   "%s: q / out rows must be 16-byte aligned and at least heads * dh wide", what);
  }
  if (a->N > 0) {
    NMTGAN_REQUIRE(a->k && a->v, "%s: null pointer", what);
    NMTGAN_REQUIRE(rows_ok(a->k, a->ldk, (int64_t)a->kv_heads * a->dh, es) && rows_ok(a->v, a->ldv, (int64_t)a->kv_heads * a->dh, es),
                   "%s: k / v rows must be 16-byte aligned and at least kv_heads * dh wide", what);
  }
  p = SpanParams{};
  p.q = a->q; p.k = a->k; p.v = a->v; p.ldq = a->ldq; p.ldk = a->ldk; p.ldv = a->ldv; p.ldo = a->ldo;
  p.lo = a->lo; p.hi = a->hi; p.pos = a->pos; p.slopes = a->slopes; p.out = a->out; p.lse = a->lse;
  p.M = a->M; p.N = a->N; p.heads = a->heads; p.kv_heads = a->kv_heads; p.dh = a->dh;
  p.scale = a->scale; p.cap = a->cap;
  return 0;
}

int launch_attn_span(const nmtgan_span_args* a, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  SpanParams p;
  NMTGAN_TRY(fill_span(a, p, "attn_span"));
  if (p.M == 0) return 0;
  NMTGAN_DISPATCH_OP(a->dtype, T, hipLaunchKernelGGL(span_fwd_rows_kernel<T>, dim3((p.M + 3) / 4, p.heads), dim3(256), 0, st, p));
  NMTGAN_CHECK_LAUNCH("attn_span");
  return 0;
}

// Workgroups along a span: enough to fill the chip, none with less than 256 keys.  max_keys is a hint (the split is
// made of the true length on the device), so a wrong one costs time only.
static int span_splits(int M, int kv_heads, int max_keys) {
  const int64_t groups = std::max<int64_t>(1, (int64_t)M * kv_heads);
  const int64_t fill = (1024 + groups - 1) / groups;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(fill, 64), (max_keys + 255) / 256));
}
size_t attn_span_step_workspace(int M, int heads, int kv_heads, int dh, int max_keys) {
  if (M <= 0 || heads <= 0 || kv_heads <= 0 || dh <= 0) return 0;
  return (size_t)M * heads * span_splits(M, kv_heads, max_keys) * (dh + 2) * sizeof(float);
}
int launch_attn_span_step(const nmtgan_span_args* a, int max_keys, void* ws, size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  SpanParams p;
  NMTGAN_TRY(fill_span(a, p, "attn_span_step"));
  NMTGAN_REQUIRE(max_keys >= 0, "attn_span_step: max_keys=%d", max_keys);
  if (p.M == 0) return 0;
  const size_t need = attn_span_step_workspace(p.M, p.heads, p.kv_heads, p.dh, max_keys);
  NMTGAN_REQUIRE(ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0, "attn_span_step: workspace of %zu bytes needed, %zu given",
                 need, ws_bytes);
  const int splits = span_splits(p.M, p.kv_heads, max_keys);
  NMTGAN_REQUIRE((int64_t)p.M * splits < (1LL << 31), "attn_span_step: too many rows");
  NMTGAN_DISPATCH_OP(a->dtype, T, {
    hipLaunchKernelGGL(span_step_kernel<T>, dim3(p.M * splits, p.heads), dim3(256), 0, st, p, splits, (float*)ws);
    NMTGAN_CHECK_LAUNCH("attn_span_step");
    hipLaunchKernelGGL(span_join_kernel<T>, dim3((unsigned)(((int64_t)p.M * p.heads + 3) / 4)), dim3(256), 0, st, p, splits,
                       (const float*)ws);
  });
  NMTGAN_CHECK_LAUNCH("attn_span_join");
  return 0;
}

static size_t carve_span_grads(int M, int heads, char* base, float** delta, int2** hull) {
  const size_t a = align_up((size_t)M * heads * sizeof(float), 256);
  if (base) { *delta = (float*)base; *hull = (int2*)(base + a); }
  return a + align_up((size_t)((M + 63) / 64) * sizeof(int2), 256);
}
size_t attn_span_grads_workspace(int M, int heads) {
  return M > 0 && heads > 0 ? carve_span_grads(M, heads, nullptr, nullptr, nullptr) : 0;
}
int launch_attn_span_grads(const nmtgan_span_args* a, const nmtgan_span_grads* g, void* ws, size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  SpanParams p;
  NMTGAN_TRY(fill_span(a, p, "attn_span_grads"));
  NMTGAN_REQUIRE(g != nullptr, "attn_span_grads: null gradients");
  NMTGAN_REQUIRE(a->dtype != NMTGAN_F16, "attn_span_grads: bf16 or fp32 (fp16 gradients would underflow without loss scaling)");
  const int es = dtype_size(a->dtype);
  const int64_t wq = (int64_t)p.heads * p.dh, wk = (int64_t)p.kv_heads * p.dh;
  if (p.M > 0) {
    NMTGAN_REQUIRE(p.lse && g->dout && g->dq, "attn_span_grads: null pointer");
    NMTGAN_REQUIRE(rows_ok(g->dout, g->ld_dout, wq, es) && rows_ok(g->dq, g->ld_dq, wq, es),
                   "attn_span_grads: dout / dq rows must be 16-byte aligned and at least heads * dh wide");
  }
  if (p.N > 0) {
    NMTGAN_REQUIRE(g->dk && g->dv, "attn_span_grads: null pointer");
    NMTGAN_REQUIRE(rows_ok(g->dk, g->ld_dk, wk, es) && rows_ok(g->dv, g->ld_dv, wk, es),
                   "attn_span_grads: dk / dv rows must be 16-byte aligned and at least kv_heads * dh wide");
  }
  const size_t need = attn_span_grads_workspace(p.M, p.heads);
  NMTGAN_REQUIRE(need == 0 || (ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0),
                 "attn_span_grads: workspace of %zu bytes needed, %zu given", need, ws_bytes);
  if (p.M > 0) carve_span_grads(p.M, p.heads, (char*)ws, &p.delta, &p.hull);
  p.dout = g->dout; p.ld_do = g->ld_dout; p.dq = g->dq; p.dk = g->dk; p.dv = g->dv;
  p.ld_dq = g->ld_dq; p.ld_dk = g->ld_dk; p.ld_dv = g->ld_dv;
  NMTGAN_DISPATCH_OP(a->dtype == NMTGAN_BF16 ? NMTGAN_BF16 : NMTGAN_F32, T, {
    if (p.M > 0) {
      hipLaunchKernelGGL(span_prep_kernel<T>, dim3((p.M + 63) / 64), dim3(256), 0, st, p);
      NMTGAN_CHECK_LAUNCH("attn_span_prep");
      hipLaunchKernelGGL(span_dq_rows_kernel<T>, dim3((p.M + 3) / 4, p.heads), dim3(256), 0, st, p);
      NMTGAN_CHECK_LAUNCH("attn_span_dq");
    }
    if (p.N > 0) {
      hipLaunchKernelGGL(span_dkv_keys_kernel<T>, dim3((p.N + 3) / 4, p.kv_heads), dim3(256), 0, st, p);
      NMTGAN_CHECK_LAUNCH("attn_span_dkv");
    }
  });
  return 0;
}

}  // namespace nmtgan
