// Softmax cross entropy of hidden rows against a vocabulary table, logits never in memory (and its gradient, d(logits)
// one piece of the vocabulary at a time):
//   z = h w^T    q_label = 1 - eps, q_j = eps / (V - 1) elsewhere
//   loss_i = lse_i - sum_j q_j z_ij = lse_i - high z_label - low sum_j z_ij        low = eps / (V - 1), high = 1 - eps - low
//   dz_ij = g_i (exp(z_ij - lse_i) - q_j)      dh = dz w      dw = dz^T h
// Rows whose label lies outside [0, V) have loss 0 and no gradient.
//
// Forward: one product on the matrix cores whose epilogue leaves (max, sum exp) per 64 entries and row (gemm.hip), joined
// in tile order by xent_finish_kernel, which also forms the label's own logit from the operands.
// Gradient, per piece of the vocabulary: the product again (2 M V d operations are cheaper at d <= 1024 than 8 bytes of
// fp32 logit written and read), its epilogue writes dz in the operand type, entry-major; two products with that image give
// the piece's rows of dw (K = rows) and partials of dh (K = entries, both operands turned on their way out of LDS).  dz is
// rounded once to the operand type - the matrix cores take no more - like every activation gradient of this library; lse,
// loss and all sums are fp32.
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.h"
#include "kernels.h"

namespace nmtgan {

__device__ __forceinline__ float xexp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// A workgroup = 16 rows x 16 groups of vocabulary tiles; groups are joined in order through LDS.  The label's logit is
// a dot product of 16 lanes per row over the same operands the matrix cores read.
template <typename T>
__global__ __launch_bounds__(256) void xent_finish_kernel(const float2* stats, const float* zsum, int n_tiles, const T* h,
                                                          int64_t ldh, const T* w, int64_t ldw, const int32_t* labels, int M,
                                                          int V, int d, float low, float high, float* loss, float* lse) {
  __shared__ float sm[16][17], ss[16][17], sz[16][17];
  const int rr = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int r = min(blockIdx.x * 16 + rr, M - 1);
  const int t0 = (int)((int64_t)n_tiles * q / 16), t1 = (int)((int64_t)n_tiles * (q + 1) / 16);
  float m = -INFINITY, s = 0.f, z = 0.f;
  for (int t = t0; t < t1; ++t) {
    const float2 a = stats[(int64_t)t * M + r];
    const float mn = fmaxf(m, a.x), mu = mn == -INFINITY ? 0.f : mn;
    s = s * xexp(m - mu) + a.y * xexp(a.x - mu);
    m = mn;
    if (zsum) z += zsum[(int64_t)t * M + r];
  }
  sm[rr][q] = m;
  ss[rr][q] = s;
  sz[rr][q] = z;
  __syncthreads();
  // from here on 16 lanes per row: row r2, lane c
  const int r2 = threadIdx.x >> 4, c = threadIdx.x & 15, row = blockIdx.x * 16 + r2;
  if (row >= M) return;
  const int label = labels[row];
  const bool used = label >= 0 && label < V;
  float dot = 0.f;
  if (used) {
    const T* hr = h + row * ldh;
    const T* wr = w + label * ldw;
    for (int k = 8 * c; k < d; k += 128) {
      float a[8], b[8];
      if (k + 8 <= d) {
        VecIO<T, 8>::load(hr + k, a);
        VecIO<T, 8>::load(wr + k, b);
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(a[e], b[e], dot);
      } else {
        for (int e = k; e < d; ++e) dot = fmaf(OpTraits<T>::load(hr + e), OpTraits<T>::load(wr + e), dot);
      }
    }
  }
  dot = dpp_add<0xB1>(dot);
  dot = dpp_add<0x4E>(dot);
  dot = dpp_add<0x141>(dot);
  dot = dpp_add<0x140>(dot);
  if (c == 0) {
    float mt = -INFINITY;
    for (int k = 0; k < 16; ++k) mt = fmaxf(mt, sm[r2][k]);
    const float mu = mt == -INFINITY ? 0.f : mt;
    float st = 0.f, zt = 0.f;
    for (int k = 0; k < 16; ++k) {
      st += ss[r2][k] * xexp(sm[r2][k] - mu);
      zt += sz[r2][k];
    }
    const float ls = mu + logf(st);
    lse[row] = ls;
    float v = ls - high * dot;
    if (zsum) v -= low * zt;
    loss[row] = used ? v : 0.f;
  }
}

// out[c][r] = in[r][c] for r < R, 0 for R <= r < Rp; rows whose label names no entry count as zeros (labels may be null)
template <typename T>
__global__ __launch_bounds__(256) void xent_transpose_kernel(const T* in, int64_t ld, int R, int C, T* out, int Rp,
                                                             const int32_t* labels, int V) {
  __shared__ T tile[64][66];
  const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + ty + 4 * i, c = c0 + tx;
    T v = T(0);
    if (r < R && c < C && (!labels || (labels[r] >= 0 && labels[r] < V))) v = in[(int64_t)r * ld + c];
    tile[ty + 4 * i][tx] = v;
  }
  __syncthreads();
  for (int i = 0; i < 16; ++i) {
    const int c = c0 + ty + 4 * i, r = r0 + tx;
    if (c < C && r < Rp) out[(int64_t)c * Rp + r] = tile[tx][ty + 4 * i];
  }
}

// per-row operands of the d(logits) epilogue, padded: coef = gradient of the row's loss (0 without a label), lse / ln 2, label
__global__ __launch_bounds__(256) void xent_rows_kernel(const int32_t* labels, const float* grad_row, const float* lse, int M,
                                                        int Mp, int V, float* coef, float* lse2, int32_t* label) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= Mp) return;
  const bool used = r < M && labels[r] >= 0 && labels[r] < V;
  coef[r] = used ? (grad_row ? grad_row[r] : 1.f) : 0.f;
  lse2[r] = r < M ? lse[r] * 1.44269504088896341f : 0.f;
  label[r] = used ? labels[r] : -1;
}

// Column sums behind label smoothing, whose constant -coef_r low of every d(logit) is kept out of the 16-bit images:
// dh_r -= coef_r low sum_j w_j, dw_j -= low sum_r coef_r h_r.  part[block][d] = sums over a block's rows (weighted if coef
// is given), added in block order by xent_colsum_finish_kernel.
constexpr int COLSUM_BLOCKS = 256;
template <typename T>
__global__ __launch_bounds__(256) void xent_colsum_kernel(const T* x, int64_t ld, int R, int C, const float* coef, float* part) {
  __shared__ float red[4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int r0 = (int)((int64_t)R * blockIdx.x / COLSUM_BLOCKS), r1 = (int)((int64_t)R * (blockIdx.x + 1) / COLSUM_BLOCKS);
  for (int c0 = 0; c0 < C; c0 += 512) {            // 64 lanes x 8 columns, four rows at a time
    const int c = c0 + 8 * tx;
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < C)
      for (int r = r0 + ty; r < r1; r += 4) {
        const float f = coef ? coef[r] : 1.f;
        if (f == 0.f) continue;
#pragma unroll
        for (int h = 0; h < 8; h += 16 / (int)sizeof(T)) {
          if (c + h >= C) break;
          float v[16 / (int)sizeof(T)];
          VecIO<T, 16 / (int)sizeof(T)>::load(x + (int64_t)r * ld + c + h, v);
#pragma unroll
          for (int e = 0; e < 16 / (int)sizeof(T); ++e) s[h + e] = fmaf(f, v[e], s[h + e]);
        }
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      __syncthreads();
      red[ty][tx] = s[e];
      __syncthreads();
      if (ty == 0 && c + e < C) part[(int64_t)blockIdx.x * C + c + e] = (red[0][tx] + red[1][tx]) + (red[2][tx] + red[3][tx]);
    }
  }
}
__global__ __launch_bounds__(256) void xent_colsum_finish_kernel(const float* part, int C, float f, float* out) {
  __shared__ float red[4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx;
  float s = 0.f;
  if (c < C)
    for (int k = ty; k < COLSUM_BLOCKS; k += 4) s += part[(int64_t)k * C + c];
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < C) out[c] = f * ((red[0][tx] + red[1][tx]) + (red[2][tx] + red[3][tx]));
}

// dh = sum of the partials in order (+ the smoothing constant's part), rounded once
template <typename T>
__global__ __launch_bounds__(256) void xent_dh_kernel(const float* part, int n_part, int M, int d, const float* coef,
                                                      const float* wsum, T* dh, int64_t ld) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, n = (int64_t)M * d;      // d % 4 == 0
  if (i >= n) return;
  const int64_t r = i / d;
  const int c = (int)(i % d);
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < n_part; ++k) {
    float v[4];
    VecIO<float, 4>::load(part + k * n + i, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += v[e];
  }
  const float f = coef[r];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (wsum) s[e] = fmaf(f, wsum[c + e], s[e]);
    if (f == 0.f) s[e] = 0.f;
  }
  VecIO<T, 4>::store(dh + r * ld + c, s);
}

template <typename T>
__global__ __launch_bounds__(256) void xent_zero_rows_kernel(T* out, int64_t ld, int R, int C) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < (int64_t)R * C) out[(i / C) * ld + i % C] = T(0);
}

// ------------------------------------------------------------------------------------------ host
static int check_xent(const nmtgan_xent_args* a, const char* what) {
  NMTGAN_REQUIRE(a != nullptr, "%s: null args", what);
  NMTGAN_REQUIRE(valid_op_dtype(a->dtype), "%s: bad dtype %d", what, a->dtype);
  NMTGAN_REQUIRE(a->M >= 0 && a->V > 0 && a->d > 0, "%s: bad shape M=%d V=%d d=%d", what, a->M, a->V, a->d);
  const int es = dtype_size(a->dtype);
  NMTGAN_REQUIRE((int64_t)a->d * es % 16 == 0, "%s: d*esize must be a multiple of 16 bytes (d=%d)", what, a->d);
  NMTGAN_REQUIRE(a->smoothing >= 0.f && a->smoothing < 1.f && (a->smoothing == 0.f || a->V > 1),
                 "%s: smoothing must be in [0, 1), and 0 for a vocabulary of one", what);
  NMTGAN_REQUIRE(a->M == 0 || (a->h && a->labels), "%s: null pointer", what);
  NMTGAN_REQUIRE(a->w, "%s: null pointer", what);
  NMTGAN_REQUIRE(((uintptr_t)a->w % 16) == 0 && a->ldw >= a->d && a->ldw * es % 16 == 0, "%s: w rows must be 16-byte aligned", what);
  NMTGAN_REQUIRE(a->M == 0 || (((uintptr_t)a->h % 16) == 0 && a->ldh >= a->d && a->ldh * es % 16 == 0),
                 "%s: h rows must be 16-byte aligned", what);
  return 0;
}
static int pad64(int n) { return (n + 63) / 64 * 64; }

struct XentPlan {
  int rows_padded, piece, n_pieces, slices, kt_slice;        // a piece = slices of kt_slice k-tiles of 64 entries
  size_t bytes;
  float *coef, *lse2, *part, *colsum, *wsum, *hsum;
  int32_t* label;
  void *g, *gt, *wt, *ht;
};
// Pieces of the vocabulary: as few as keep a piece's d(logits) inside the 256 MB memory-side cache (the two products read
// what the epilogue wrote).  Inside a piece the hidden gradient's product is cut along the entries into enough slices to
// give every CU a tile.
static void carve_xent(const nmtgan_xent_args* a, char* base, size_t cap, XentPlan& q) {
  const int es = dtype_size(a->dtype);
  const bool f32 = a->dtype == NMTGAN_F32;
  q.rows_padded = pad64(a->M);
  const int64_t fit = (224LL << 20) / ((f32 ? 2LL : 1LL) * es * q.rows_padded);
  int64_t n = (a->V + fit - 1) / std::max<int64_t>(fit, 1);
  n = std::max<int64_t>(1, std::min<int64_t>(n, (a->V + 1023) / 1024));
  const int64_t want = (a->V + n - 1) / n, kt = std::max<int64_t>(4, (want + 63) / 64);
  const int64_t tiles = (int64_t)((a->M + 255) / 256) * (f32 ? (a->d + 127) / 128 : (a->d + 255) / 256);
  q.slices = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(24, 256 / tiles), kt / 4));
  q.kt_slice = (int)((kt + q.slices - 1) / q.slices);
  q.piece = q.slices * q.kt_slice * 64;
  q.n_pieces = (a->V + q.piece - 1) / q.piece;
  Arena ar(base, cap);
  q.coef = ar.get<float>(q.rows_padded);
  q.lse2 = ar.get<float>(q.rows_padded);
  q.label = ar.get<int32_t>(q.rows_padded);
  q.gt = ar.take((size_t)q.piece * q.rows_padded * es);
  q.ht = ar.take((size_t)a->d * q.rows_padded * es);
  q.part = ar.get<float>((size_t)q.n_pieces * q.slices * a->M * a->d);
  q.colsum = q.wsum = q.hsum = nullptr;
  if (a->smoothing > 0.f) {
    q.colsum = ar.get<float>((size_t)COLSUM_BLOCKS * a->d);
    q.wsum = ar.get<float>(a->d);
    q.hsum = ar.get<float>(a->d);
  }
  q.g = q.wt = nullptr;
  if (f32) {
    q.g = ar.take((size_t)a->M * q.piece * es);
    q.wt = ar.take((size_t)a->d * q.piece * es);
  }
  q.bytes = ar.off;
}
size_t linear_xent_workspace(const nmtgan_xent_args* a, bool grads) {
  if (!a || a->M <= 0 || a->V <= 0 || a->d <= 0 || !valid_op_dtype(a->dtype)) return 0;
  if (!grads) {
    const size_t n = (size_t)((a->V + 63) / 64) * a->M;
    return align_up(n * sizeof(float2), 256) + (a->smoothing > 0.f ? n * sizeof(float) : 0);
  }
  XentPlan q;
  carve_xent(a, nullptr, 0, q);
  return q.bytes;
}

int launch_linear_xent(const nmtgan_xent_args* a, float* loss, float* lse, void* ws, size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  NMTGAN_TRY(check_xent(a, "linear_xent"));
  if (a->M == 0) return 0;
  NMTGAN_REQUIRE(loss && lse, "linear_xent: null output");
  const size_t need = linear_xent_workspace(a, false);
  NMTGAN_REQUIRE(ws && ws_bytes >= need && (uintptr_t)ws % 256 == 0, "linear_xent: workspace of %zu bytes (256-byte aligned) needed, %zu given",
                 need, ws_bytes);
  const int tiles = (a->V + 63) / 64;
  float2* stats = (float2*)ws;
  XentEpilogue x{};
  if (a->smoothing > 0.f) x.zsum = (float*)((char*)ws + align_up((size_t)tiles * a->M * sizeof(float2), 256));
  NMTGAN_TRY(launch_gemm_xent(a->dtype, false, a->w, a->ldw, a->V, a->h, a->ldh, a->M, a->d, stats, x, st));
  const float low = a->smoothing > 0.f ? a->smoothing / (float)(a->V - 1) : 0.f, high = 1.f - a->smoothing - low;
  NMTGAN_DISPATCH_OP(a->dtype, T,
                     hipLaunchKernelGGL(xent_finish_kernel<T>, dim3((a->M + 15) / 16), dim3(256), 0, st, stats, x.zsum, tiles,
                                        (const T*)a->h, a->ldh, (const T*)a->w, a->ldw, a->labels, a->M, a->V, a->d, low, high,
                                        loss, lse));
  NMTGAN_CHECK_LAUNCH("linear_xent_finish");
  return 0;
}

template <typename T>
static int xent_grads_t(const nmtgan_xent_args* a, const float* lse, const float* grad_row, void* dh, int64_t ld_dh, void* dw,
                        int64_t ld_dw, void* ws, size_t ws_bytes, hipStream_t st) {
  constexpr int es = sizeof(T);
  if (a->M == 0) {
    hipLaunchKernelGGL(xent_zero_rows_kernel<T>, dim3((unsigned)(((int64_t)a->V * a->d + 255) / 256)), dim3(256), 0, st, (T*)dw,
                       ld_dw, a->V, a->d);
    NMTGAN_CHECK_LAUNCH("linear_xent_zero");
    return 0;
  }
  XentPlan q;
  carve_xent(a, (char*)ws, ws_bytes, q);
  const float low = a->smoothing > 0.f ? a->smoothing / (float)(a->V - 1) : 0.f;
  hipLaunchKernelGGL(xent_rows_kernel, dim3((q.rows_padded + 255) / 256), dim3(256), 0, st, a->labels, grad_row, lse, a->M,
                     q.rows_padded, a->V, q.coef, q.lse2, q.label);
  NMTGAN_CHECK_LAUNCH("linear_xent_rows");
  hipLaunchKernelGGL(xent_transpose_kernel<T>, dim3(q.rows_padded / 64, (a->d + 63) / 64), dim3(256), 0, st, (const T*)a->h,
                     a->ldh, a->M, a->d, (T*)q.ht, q.rows_padded, a->labels, a->V);
  NMTGAN_CHECK_LAUNCH("linear_xent_transpose");
  if (low > 0.f) {
    hipLaunchKernelGGL(xent_colsum_kernel<T>, dim3(COLSUM_BLOCKS), dim3(256), 0, st, (const T*)a->w, a->ldw, a->V, a->d,
                       (const float*)nullptr, q.colsum);
    NMTGAN_CHECK_LAUNCH("linear_xent_colsum");
    hipLaunchKernelGGL(xent_colsum_finish_kernel, dim3((a->d + 63) / 64), dim3(256), 0, st, q.colsum, a->d, -low, q.wsum);
    NMTGAN_CHECK_LAUNCH("linear_xent_colsum");
    hipLaunchKernelGGL(xent_colsum_kernel<T>, dim3(COLSUM_BLOCKS), dim3(256), 0, st, (const T*)a->h, a->ldh, a->M, a->d, q.coef,
                       q.colsum);
    NMTGAN_CHECK_LAUNCH("linear_xent_colsum");
    hipLaunchKernelGGL(xent_colsum_finish_kernel, dim3((a->d + 63) / 64), dim3(256), 0, st, q.colsum, a->d, -low, q.hsum);
    NMTGAN_CHECK_LAUNCH("linear_xent_colsum");
  }
  XentEpilogue x{};
  x.coef = q.coef; x.lse2 = q.lse2; x.label = q.label; x.g = q.g; x.gt = q.gt;
  x.rows_padded = q.rows_padded;
  x.piece_padded = q.piece;
  x.high = 1.f - a->smoothing - low;
  int n_part = 0;
  for (int v0 = 0; v0 < a->V; v0 += q.piece) {
    const int n = std::min(q.piece, a->V - v0);
    x.first = v0;
    const T* w = (const T*)a->w + (int64_t)v0 * a->ldw;
    NMTGAN_TRY(launch_gemm_xent(a->dtype, true, w, a->ldw, n, a->h, a->ldh, a->M, a->d, nullptr, x, st));
    float* part = q.part + (int64_t)n_part * a->M * a->d;
    if constexpr (es == 2) {
      NMTGAN_TRY(launch_gemm_kmajor(a->dtype, q.gt, q.rows_padded, q.piece, w, a->ldw, n, a->M, a->d, q.slices, q.kt_slice, part,
                                    st));
      n_part += q.slices;
    } else {
      hipLaunchKernelGGL(xent_transpose_kernel<T>, dim3(q.piece / 64, (a->d + 63) / 64), dim3(256), 0, st, w, a->ldw, n, a->d,
                         (T*)q.wt, q.piece, (const int32_t*)nullptr, 0);
      NMTGAN_CHECK_LAUNCH("linear_xent_transpose");
      nmtgan_gemm_args g[24];
      for (int s = 0; s < q.slices; ++s) {
        nmtgan_gemm_args& b = g[s];
        b = nmtgan_gemm_args{};
        b.op_dtype = a->dtype;
        b.epilogue = NMTGAN_EPI_LINEAR;
        b.A = (const T*)q.g + s * q.kt_slice * 64; b.lda = q.piece;
        b.Wt = (const T*)q.wt + s * q.kt_slice * 64; b.ldw = q.piece;
        b.M = a->M; b.N = a->d; b.K = q.kt_slice * 64;
        b.n_seg = 1; b.out[0] = part + (int64_t)s * a->M * a->d; b.ldo[0] = a->d; b.out_f32[0] = 1; b.seg_scale[0] = 1.f;
      }
      NMTGAN_TRY(launch_gemm_group(g, q.slices, st));
      n_part += q.slices;
    }
    nmtgan_gemm_args b{};
    b.op_dtype = a->dtype;
    b.epilogue = NMTGAN_EPI_LINEAR;
    b.A = q.gt; b.lda = q.rows_padded; b.Wt = q.ht; b.bias = q.hsum;
    b.M = n; b.N = a->d; b.K = q.rows_padded;
    b.n_seg = 1; b.out[0] = (T*)dw + (int64_t)v0 * ld_dw; b.ldo[0] = ld_dw; b.out_f32[0] = es == 4; b.seg_scale[0] = 1.f;
    NMTGAN_TRY(launch_gemm(&b, st));
  }
  hipLaunchKernelGGL(xent_dh_kernel<T>, dim3((unsigned)(((int64_t)a->M * a->d / 4 + 255) / 256)), dim3(256), 0, st, q.part, n_part,
                     a->M, a->d, q.coef, q.wsum, (T*)dh, ld_dh);
  NMTGAN_CHECK_LAUNCH("linear_xent_dh");
  return 0;
}
int launch_linear_xent_grads(const nmtgan_xent_args* a, const float* lse, const float* grad_row, void* dh, int64_t ld_dh,
                             void* dw, int64_t ld_dw, void* ws, size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  NMTGAN_TRY(check_xent(a, "linear_xent_grads"));
  NMTGAN_REQUIRE(a->dtype != NMTGAN_F16, "linear_xent_grads: bf16 or fp32 (fp16 gradients would underflow without loss scaling)");
  const int es = dtype_size(a->dtype);
  NMTGAN_REQUIRE(dw && (uintptr_t)dw % 16 == 0 && ld_dw >= a->d && ld_dw * es % 16 == 0, "linear_xent_grads: bad dw");
  NMTGAN_REQUIRE(a->M == 0 || (lse && dh && (uintptr_t)dh % 16 == 0 && ld_dh >= a->d && ld_dh * es % 16 == 0),
                 "linear_xent_grads: null lse or bad dh");
  const size_t need = linear_xent_workspace(a, true);
  NMTGAN_REQUIRE(need == 0 || (ws && ws_bytes >= need && (uintptr_t)ws % 256 == 0),
                 "linear_xent_grads: workspace of %zu bytes (256-byte aligned) needed, %zu given", need, ws_bytes);
  if (a->dtype == NMTGAN_BF16) return xent_grads_t<bf16_t>(a, lse, grad_row, dh, ld_dh, dw, ld_dw, ws, ws_bytes, st);
  return xent_grads_t<float>(a, lse, grad_row, dh, ld_dh, dw, ld_dw, ws, ws_bytes, st);
}

}  // namespace nmtgan
