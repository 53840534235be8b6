// Span attention: preparation of the gradients, the form for single tokens, checks and launches (span_tiles.h has the formulas).
#include "span_tiles.h"

namespace nmtgan {

// What the gradient kernels need per row and per 32 rows: delta_i = dout_i . out_i of every head (0 for rows that see
// nothing, whatever their dout holds) and
// the hull of the spans of 32 rows.  One workgroup per 64 rows; a row's head products are
// summed by 8 lanes.
template <typename T>
__global__ __launch_bounds__(256) void span_prep_kernel(SpanParams p) {
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (w == 0) {
    const int i = b * 64 + lane;
    int2 sp = make_int2(0, 0);
    if (i < p.M) sp = span_of(p, i);
    int4 hl = make_int4(sp.y > sp.x ? sp.x : 0x7fffffff, sp.y, sp.x, sp.y);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      hl.x = min(hl.x, __shfl_xor(hl.x, o, 64));
      hl.y = max(hl.y, __shfl_xor(hl.y, o, 64));
      hl.z = max(hl.z, __shfl_xor(hl.z, o, 64));
      hl.w = min(hl.w, __shfl_xor(hl.w, o, 64));
    }
    if ((lane & 31) == 0 && i < p.M) p.hull[2 * b + (lane >> 5)] = hl;
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
  return span_fwd_tiles(a->dtype, p, st);
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

static size_t carve_span_grads(int M, int heads, char* base, float** delta, int4** hull) {
  const size_t a = align_up((size_t)M * heads * sizeof(float), 256);
  if (base) { *delta = (float*)base; *hull = (int4*)(base + a); }
  return a + align_up((size_t)((M + 31) / 32) * sizeof(int4), 256);
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
  if (p.M > 0) {
    NMTGAN_DISPATCH_GRAD(a->dtype, T, hipLaunchKernelGGL(span_prep_kernel<T>, dim3((p.M + 63) / 64), dim3(256), 0, st, p));
    NMTGAN_CHECK_LAUNCH("attn_span_prep");
    NMTGAN_TRY(span_dq_tiles(a->dtype, p, st));
  }
  return p.N > 0 ? span_dkv_tiles(a->dtype, p, st) : 0;
}

}  // namespace nmtgan
