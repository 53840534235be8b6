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
// fp32 logit written and read), its epilogue writes the image y = p / high - [j = label] in the operand type, entry-major;
// two products with it give the piece's rows of dw = high y^T (g h) + ... (K = rows) and partials of dh = g high (y w) + ...
// (K = entries, both operands turned on their way out of LDS).  y and g h are rounded once to the operand type - the matrix
// cores take no more - like every activation gradient of this library; lse, loss and all sums are fp32.  Neither g nor high
// is in y: where all rows weigh the same, g high is one number in every row, and its rounding would add up over them
// (3200 rows of 1 / 3200 over 32000 entries, smoothing 0.1: error of dh and dw 0.0035 of their size with it, 0.0023
// without).  The label's
// -1 is exact.
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.h"
#include "kernels.h"
#include "regions.h"

namespace nmtgan {

__device__ __forceinline__ float xexp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// A workgroup = 16 rows x 16 groups of vocabulary tiles; groups are joined in order through LDS.  The label's logit is
// a dot product of 16 lanes per row over the same operands the matrix cores read.  Bound by the latency of its few dependent
// loads: 3200 rows x 500 tiles with smoothing (19 MB) 11.8 us, 1601 rows without 8 us.
template <typename T>
__global__ __launch_bounds__(256) void xent_finish_kernel(const float2* stats, const float* zsum, int n_tiles, const T* h,
                                                          int64_t ldh, const T* w, int64_t ldw, const int32_t* labels, int M,
                                                          int V, int d, float low, float high, float* loss, float* lse) {
  __shared__ float sm[16][17], ss[16][17], sz[16][17];
  const int rr = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int r = min(blockIdx.x * 16 + rr, M - 1);
  const int t0 = (int)((int64_t)n_tiles * q / 16), t1 = (int)((int64_t)n_tiles * (q + 1) / 16);
  float m = -INFINITY, s = 0.f, z = 0.f;
  for (int t = t0; t < t1; t += 8) {                         // eight tiles in flight
    float2 a[8];
    float zs[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      a[k] = t + k < t1 ? stats[(int64_t)(t + k) * M + r] : make_float2(-INFINITY, 0.f);
      zs[k] = zsum && t + k < t1 ? zsum[(int64_t)(t + k) * M + r] : 0.f;
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) mn = fmaxf(mn, a[k].x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    s *= xexp(m - mu);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      s = fmaf(a[k].y, xexp(a[k].x - mu), s);
      z += zs[k];
    }
    m = mn;
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

// out[c][r] = row(r, c), a function that is 0 outside the input, for r < Rp and c < C: one 64 x 64 tile
template <typename T, typename Row>
__device__ __forceinline__ void transpose_tile(T (&tile)[64][66], Row row, int C, T* out, int Rp, int r0, int c0) {
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    tile[ty + 4 * i][tx] = row(r0 + ty + 4 * i, c0 + tx);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int c = c0 + ty + 4 * i, r = r0 + tx;
    if (c < C && r < Rp) out[(int64_t)c * Rp + r] = tile[tx][ty + 4 * i];
  }
}
// Everything the gradient needs before its first product, in one launch by roles of workgroups:
//   - per row, padded: coef = gradient of the row's loss (0 without a label), factor = 1 / unit (0 where coef is), lse / ln 2,
//     label.  unit = high, or 1 where the smoothing leaves high = 0
//   - (coef h)^T, zero in rows without a label and in the padding
//   - column sums behind label smoothing, whose constant -coef_r low of every d(logit) is kept out of the 16-bit images:
//     dh_r -= coef_r low sum_j w_j, dw_j -= low sum_r coef_r h_r.  part[block][d], added in block order afterwards
// (3200 rows, 32000 entries, d = 512: 14 to 18 us for 36 MB)
constexpr int SUM_W = 256, SUM_H = 128;
struct XentPrep {
  const void* h; const void* w; int64_t ldh, ldw;
  const int32_t* labels; const float* grad_row; const float* lse;
  float* coef; float* factor; float* lse2; int32_t* label;
  void* ht; float* part;
  float inv_unit;
  int M, Mp, V, d, n_rows, n_turn;                 // workgroups of the first two roles
};
__device__ __forceinline__ float row_coef(const XentPrep& p, int r) {
  const bool used = p.labels[r] >= 0 && p.labels[r] < p.V;
  return used ? (p.grad_row ? p.grad_row[r] : 1.f) : 0.f;
}
template <typename T>
__global__ __launch_bounds__(256) void xent_prep_kernel(XentPrep p) {
  __shared__ T tile[64][66];
  __shared__ float red[4][64];
  int b = blockIdx.x;
  if (b < p.n_rows) {
    const int r = b * 256 + threadIdx.x;
    if (r >= p.Mp) return;
    const bool used = r < p.M && p.labels[r] >= 0 && p.labels[r] < p.V;
    const float coef = r < p.M ? row_coef(p, r) : 0.f;
    p.coef[r] = coef;
    p.factor[r] = coef == 0.f ? 0.f : p.inv_unit;
    p.lse2[r] = r < p.M ? p.lse[r] * 1.44269504088896341f : 0.f;
    p.label[r] = used ? p.labels[r] : -1;
    return;
  }
  b -= p.n_rows;
  if (b < p.n_turn) {
    const int across = p.Mp / 64;
    auto row = [&](int r, int c) {
      const float g = r < p.M ? row_coef(p, r) : 0.f;
      T v = T(0);
      if (g != 0.f && c < p.d) OpTraits<T>::store(&v, g * OpTraits<T>::load((const T*)p.h + (int64_t)r * p.ldh + c));
      return v;
    };
    transpose_tile<T>(tile, row, p.d, (T*)p.ht, p.Mp, b % across * 64, b / across * 64);
    return;
  }
  b -= p.n_turn;
  constexpr int E = 16 / (int)sizeof(T);
  const bool of_w = b < SUM_W;
  const T* x = (const T*)(of_w ? p.w : p.h);
  const int64_t ld = of_w ? p.ldw : p.ldh;
  const int R = of_w ? p.V : p.M, blk = of_w ? b : b - SUM_W, blocks = of_w ? SUM_W : SUM_H;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int r0 = (int)((int64_t)R * blk / blocks), r1 = (int)((int64_t)R * (blk + 1) / blocks);
  for (int c0 = 0; c0 < p.d; c0 += 64 * E) {       // 64 lanes x 16 bytes, four rows at a time
    const int c = c0 + E * tx;
    float s[E];
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] = 0.f;
    if (c < p.d) {
      constexpr int U = 4;
      for (int r = r0 + ty; r < r1; r += 4 * U) {
        float v[U][E], f[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          f[u] = r + 4 * u < r1 ? (of_w ? 1.f : row_coef(p, r + 4 * u)) : 0.f;
          VecIO<T, E>::load(x + (int64_t)min(r + 4 * u, r1 - 1) * ld + c, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) s[e] += f[u] == 0.f ? 0.f : f[u] * v[u][e];
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      __syncthreads();
      red[ty][tx] = s[e];
      __syncthreads();
      if (ty == 0 && c + e < p.d) p.part[(int64_t)b * p.d + c + e] = (red[0][tx] + red[1][tx]) + (red[2][tx] + red[3][tx]);
    }
  }
}
// wsum = fw sum of w's parts, hsum = fh sum of h's, 16 threads per column
__global__ __launch_bounds__(1024) void xent_sums_kernel(const float* part, int d, float fw, float fh, float* wsum, float* hsum) {
  __shared__ float red[16][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6, c = blockIdx.x * 64 + tx;
  const bool of_w = blockIdx.y == 0;
  const float* q = part + (of_w ? 0 : (int64_t)SUM_W * d);
  float s = 0.f;
  if (c < d) {
    if (of_w) {
#pragma unroll
      for (int k = 0; k < SUM_W / 16; ++k) s += q[(int64_t)(ty * (SUM_W / 16) + k) * d + c];
    } else {
#pragma unroll
      for (int k = 0; k < SUM_H / 16; ++k) s += q[(int64_t)(ty * (SUM_H / 16) + k) * d + c];
    }
  }
  red[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < d) {
    float t = 0.f;
    for (int k = 0; k < 16; ++k) t += red[k][tx];
    (of_w ? wsum : hsum)[c] = (of_w ? fw : fh) * t;
  }
}

// dh = coef (unit times the sum of the partials in order + the smoothing constant's part), rounded once; without coef the
// plain sum
template <typename T>
__global__ __launch_bounds__(256) void xent_dh_kernel(const float* part, int n_part, int M, int d, const float* coef,
                                                      float unit, const float* wsum, T* dh, int64_t ld) {
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
  const float f = coef ? coef[r] : 1.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s[e] = f == 0.f ? 0.f : f * fmaf(unit, s[e], wsum ? wsum[c + e] : 0.f);
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
  constexpr int MOST = INT32_MAX - 65536;         // indexes run over the end of the last tile
  NMTGAN_REQUIRE(a->M >= 0 && a->V > 0 && a->d > 0 && a->M <= MOST && a->V <= MOST, "%s: bad shape M=%d V=%d d=%d", what, a->M,
                 a->V, a->d);
  NMTGAN_REQUIRE((int64_t)((a->M + 127) / 128) * ((a->V + 127) / 128) < (1LL << 31), "%s: more than 2^31 tiles of 128 x 128 logits",
                 what);
  NMTGAN_REQUIRE(a->ldw <= 1 << 20 && a->ldh <= 1 << 20, "%s: rows further than 2^20 elements apart", what);
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
  int rows_padded, piece, slices, kt_slice;        // a piece = slices of kt_slice k-tiles of 64 entries
  int row_slices, kt_rows;                         // dw's k-loop: slices of kt_rows k-tiles of 64 rows
  int sets;                                        // sets of dh's partial sums that the pieces take in turn
  size_t bytes;
  float *coef, *factor, *lse2, *part, *part_w, *colsum, *wsum, *hsum;
  int32_t* label;
  void *y, *ht, *splitk;
};
constexpr size_t SPLITK_BYTES = 8 << 20;
// Pieces of the vocabulary: as few as keep a piece's d(logits) inside the 256 MB memory-side cache (the two products read
// what the epilogue wrote).
constexpr int64_t PIECE_BYTES = 224LL << 20;
static int64_t pieces_of(const nmtgan_xent_args* a, int64_t entry_bytes) {
  const int64_t fit = std::max<int64_t>(PIECE_BYTES / entry_bytes, 1);
  return std::max<int64_t>(1, std::min<int64_t>((a->V + fit - 1) / fit, (a->V + 255) / 256));
}
// Partial sums of dh are kept apart by pieces up to a gigabyte (of 288) and added to behind it: 8000 rows over 50257 entries,
// d = 1024, 262 MB of them: the product writes them in 174 us a piece and adds to them in 217.
constexpr int64_t SETS_BYTES = 1LL << 30;
// 16-bit products.  Inside a piece the hidden gradient's product is cut along the entries into enough slices to give every
// CU a tile.
static void carve_xent(const nmtgan_xent_args* a, char* base, size_t cap, XentPlan& q) {
  const int es = dtype_size(a->dtype);
  q.rows_padded = pad64(a->M);
  const int64_t n = std::max<int64_t>(pieces_of(a, (int64_t)es * q.rows_padded), (a->V * a->ldw + (1LL << 30) - 1) >> 30);   // (32-bit offsets)
  const int64_t want = (a->V + n - 1) / n, kt = std::max<int64_t>(4, (want + 63) / 64);
  const int64_t tiles = (int64_t)((a->M + 255) / 256) * ((a->d + 255) / 256);
  q.slices = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(24, 256 / tiles), kt / 4));
  q.kt_slice = (int)((kt + q.slices - 1) / q.slices);
  q.piece = q.slices * q.kt_slice * 64;
  q.sets = (int)std::max<int64_t>(1, std::min<int64_t>((a->V + q.piece - 1) / q.piece, SETS_BYTES / (4LL * q.slices * a->M * a->d)));
  // dw of a piece with few tiles and many rows: the rows are cut too (65536 rows over 32000 entries, d = 512: 109 us and 20 for
  // the sum a piece, 849 without).  Strides of a multiple of 2 KiB are avoided: rows of the
  // images would fall on a few memory channels.
  const int64_t tiles_w = (int64_t)((q.piece + 255) / 256) * ((a->d + 255) / 256);
  q.kt_rows = q.rows_padded / 64;
  q.row_slices = tiles_w < 192 ? (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(256 / tiles_w, 15), q.kt_rows / 6)) : 1;
  q.kt_rows = (q.kt_rows + q.row_slices - 1) / q.row_slices;
  while (q.row_slices * q.kt_rows % 16 == 0) ++q.kt_rows;
  q.rows_padded = 64 * q.row_slices * q.kt_rows;
  Arena ar(base, cap);
  q.coef = ar.get<float>(q.rows_padded);
  q.factor = ar.get<float>(q.rows_padded);
  q.lse2 = ar.get<float>(q.rows_padded);
  q.label = ar.get<int32_t>(q.rows_padded);
  q.y = ar.take((size_t)q.piece * q.rows_padded * es);
  q.ht = ar.take((size_t)a->d * q.rows_padded * es);
  q.part = ar.get<float>((size_t)q.sets * q.slices * a->M * a->d);
  q.part_w = q.row_slices > 1 ? ar.get<float>((size_t)q.row_slices * q.piece * a->d) : nullptr;
  q.colsum = q.wsum = q.hsum = nullptr;
  if (a->smoothing > 0.f) {
    q.colsum = ar.get<float>((size_t)(SUM_W + SUM_H) * a->d);
    q.wsum = ar.get<float>(a->d);
    q.hsum = ar.get<float>(a->d);
  }
  q.splitk = ar.take(SPLITK_BYTES);
  q.bytes = ar.off;
}
// The direct form (xent_direct.hip) against this file's products on the library's tiles, by M V d and rows:
//   logits in fp32 up to 1e9 (50 x 9000 x 256: 16 us against 39, 900 x 9000 x 128: 42 against 43), in 16 bits never (8 x
//   32000 x 512: 20 against 19);
//   gradient's products in fp32 always (97 x 509 x 64, with the logits: 13 us against 70, 900 x 9000 x 512: 480 against 1362,
//   3200 x 32000 x 512: 4.7 ms against 6.6), in 16 bits up to 3e8 (900 x 1000 x 256: 36 us against 55, 200 x 4000 x 256: 42
//   against 49, 400 x 4000 x 256: 68 against 54) and up to one tile of 32 rows, where the table's bytes count and not the
//   products (8 x 32000 x 512: 57 against 99, 8 x 50257 x 1024: 126 against 203, 32 x 50257 x 1024: 161 against 205, 32 x
//   128256 x 1024: 390 against 485; 64 rows of these two: 278 against 209, 703 against 489).
static int64_t xent_work(const nmtgan_xent_args* a) { return (int64_t)a->M * a->V * a->d; }
static bool direct_logits(const nmtgan_xent_args* a) { return a->dtype == NMTGAN_F32 && xent_work(a) <= 1000000000; }
static bool direct_grads(const nmtgan_xent_args* a) { return a->dtype == NMTGAN_F32 || a->M <= 32 || xent_work(a) <= 300000000; }
struct DirectPlan {
  XentDirect p;
  int piece, n_pieces;
  size_t bytes;
  float *factor, *lse2;                          // these and label for logits on the library's tiles only
  int32_t* label;
};
static float xent_low(const nmtgan_xent_args* a) { return a->smoothing > 0.f ? a->smoothing / (float)(a->V - 1) : 0.f; }
static XentDirect direct_params(const nmtgan_xent_args* a) {
  XentDirect p{};
  p.h = a->h; p.w = a->w; p.ldh = a->ldh; p.ldw = a->ldw;
  p.labels = a->labels;
  p.M = a->M; p.V = a->V; p.Vp = (a->V + 7) / 8 * 8; p.d = a->d;
  p.V_all = a->V;
  p.low = xent_low(a);
  p.high = 1.f - a->smoothing - p.low;
  return p;
}
// Pieces as above; dh's entries cut into slices of 1024 at least (16 waves share one) and dw's rows into slices of 2048 at
// least, no more than give every CU a workgroup
static void carve_direct(const nmtgan_xent_args* a, char* base, size_t cap, DirectPlan& q) {
  q.p = direct_params(a);
  const int64_t n = pieces_of(a, 4LL * a->M);
  q.piece = (int)((a->V + 8 * n - 1) / (8 * n) * 8);
  q.n_pieces = (a->V + q.piece - 1) / q.piece;
  const int64_t down = (a->M + 31) / 32, down_w = (q.piece + 31) / 32;
  q.p.cols = (down + down_w) * ((a->d + 63) / 64) >= 512 ? 2 : 1;
  const int64_t across = (a->d + 32 * q.p.cols - 1) / (32 * q.p.cols), tiles = down * across, tiles_w = down_w * across;
  q.p.slices = (int)std::max<int64_t>(1, std::min<int64_t>(q.piece / 1024, 256 / tiles));
  q.p.waves = tiles_w < 1024 ? 16 : (a->M > 64 ? 4 : 1);        // (1: at most eight steps)
  q.p.row_slices = (int)std::max<int64_t>(1, std::min<int64_t>(a->M / 2048, 256 * 16 / (tiles_w * q.p.waves)));
  Arena ar(base, cap);
  q.p.coef = ar.get<float>(pad64(a->M));
  q.p.y = ar.get<float>((size_t)a->M * q.piece);
  q.p.part = q.n_pieces > 1 || q.p.slices > 1 ? ar.get<float>((size_t)q.p.slices * a->M * a->d) : nullptr;
  q.p.part_w = q.p.row_slices > 1 ? ar.get<float>((size_t)q.p.row_slices * q.piece * a->d) : nullptr;
  q.factor = q.lse2 = nullptr;
  q.label = nullptr;
  if (!direct_logits(a) && a->dtype == NMTGAN_F32) {
    q.factor = ar.get<float>(pad64(a->M));
    q.lse2 = ar.get<float>(pad64(a->M));
    q.label = ar.get<int32_t>(pad64(a->M));
  }
  q.bytes = ar.off;
}
// forward: statistics per 64 entries (32 in the direct form) and row
static size_t carve_forward(const nmtgan_xent_args* a, char* base, size_t cap, int& tiles, float2*& stats, float*& zsum) {
  const int per = direct_logits(a) ? 32 : 64;
  tiles = (a->V + per - 1) / per;
  Arena ar(base, cap);
  stats = ar.get<float2>((size_t)tiles * a->M);
  zsum = a->smoothing > 0.f ? ar.get<float>((size_t)tiles * a->M) : nullptr;
  return ar.off;
}
size_t linear_xent_workspace(const nmtgan_xent_args* a, bool grads) {
  if (!a || a->M <= 0 || a->V <= 0 || a->d <= 0 || !valid_op_dtype(a->dtype)) return 0;
  if (!grads) {
    int tiles;
    float2* stats;
    float* zsum;
    return carve_forward(a, nullptr, 0, tiles, stats, zsum);
  }
  if (direct_grads(a)) {
    DirectPlan q;
    carve_direct(a, nullptr, 0, q);
    return q.bytes;
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
  const int es = dtype_size(a->dtype);
  NMTGAN_TRY(refuse_overlaps("linear_xent",
                             {Region("loss", loss, 4LL * a->M), Region("lse", lse, 4LL * a->M), Region("workspace", ws, (int64_t)need)},
                             {Region("h", a->h, a->M, a->ldh * es, (int64_t)a->d * es), Region("w", a->w, a->V, a->ldw * es, (int64_t)a->d * es),
                              Region("labels", a->labels, 4LL * a->M)}));
  int tiles;
  float2* stats;
  XentEpilogue x{};
  carve_forward(a, (char*)ws, ws_bytes, tiles, stats, x.zsum);
  if (direct_logits(a)) {
    XentDirect p = direct_params(a);
    p.stats = stats;
    p.zsum = x.zsum;
    NMTGAN_TRY(launch_xent_direct_z(a->dtype, false, p, st));
  } else {
    NMTGAN_TRY(launch_gemm_xent(a->dtype, false, a->w, a->ldw, a->V, a->h, a->ldh, a->M, a->d, stats, x, st));
  }
  const float low = xent_low(a), high = 1.f - a->smoothing - low;
  NMTGAN_DISPATCH_OP(a->dtype, T,
                     hipLaunchKernelGGL(xent_finish_kernel<T>, dim3((a->M + 15) / 16), dim3(256), 0, st, stats, x.zsum, tiles,
                                        (const T*)a->h, a->ldh, (const T*)a->w, a->ldw, a->labels, a->M, a->V, a->d, low, high,
                                        loss, lse));
  NMTGAN_CHECK_LAUNCH("linear_xent_finish");
  return 0;
}

template <typename T>
static int direct_grads_t(const nmtgan_xent_args* a, const float* lse, const float* grad_row, void* dh, int64_t ld_dh, void* dw,
                          int64_t ld_dw, void* ws, size_t ws_bytes, hipStream_t st) {
  DirectPlan q;
  carve_direct(a, (char*)ws, ws_bytes, q);
  XentDirect& p = q.p;
  p.lse = lse; p.grad_row = grad_row;
  p.dh = dh; p.ld_dh = ld_dh; p.ld_dw = ld_dw;
  if (q.factor) {
    XentPrep pr{};
    pr.labels = a->labels; pr.grad_row = grad_row; pr.lse = lse;
    pr.coef = p.coef; pr.factor = q.factor; pr.lse2 = q.lse2; pr.label = q.label;
    pr.inv_unit = 1.f;
    pr.M = a->M; pr.Mp = pad64(a->M); pr.V = a->V;
    pr.n_rows = (pr.Mp + 255) / 256;
    hipLaunchKernelGGL(xent_prep_kernel<T>, dim3(pr.n_rows), dim3(256), 0, st, pr);
    NMTGAN_CHECK_LAUNCH("linear_xent_prep");
  }
  auto sum = [&](const float* part, int n, int rows, const float* coef, T* out, int64_t ld) -> int {
    hipLaunchKernelGGL(xent_dh_kernel<T>, dim3((unsigned)(((int64_t)rows * a->d / 4 + 255) / 256)), dim3(256), 0, st, part, n,
                       rows, a->d, coef, 1.f, nullptr, out, ld);
    NMTGAN_CHECK_LAUNCH("linear_xent_sum");
    return 0;
  };
  for (int v0 = 0; v0 < a->V; v0 += q.piece) {
    p.first = v0;
    p.V = std::min(q.piece, a->V - v0);
    p.Vp = (p.V + 7) / 8 * 8;
    p.w = (const T*)a->w + (int64_t)v0 * a->ldw;
    p.dw = (T*)dw + (int64_t)v0 * ld_dw;
    p.add = v0 > 0;
    if (q.factor) {
      XentEpilogue x{};
      x.factor = q.factor; x.lse2 = q.lse2; x.label = q.label; x.y = p.y;
      x.rows_padded = pad64(a->M);
      x.piece_padded = p.Vp;
      x.first = v0;
      x.high = p.high;
      x.low = p.low;
      NMTGAN_TRY(launch_gemm_xent(a->dtype, true, p.w, a->ldw, p.V, a->h, a->ldh, a->M, a->d, nullptr, x, st));
    } else {
      NMTGAN_TRY(launch_xent_direct_z(a->dtype, true, p, st));
    }
    NMTGAN_TRY(launch_xent_direct_grads(a->dtype, p, st));
    if (p.part_w) NMTGAN_TRY(sum(p.part_w, p.row_slices, p.V, nullptr, (T*)p.dw, ld_dw));
  }
  if (p.part) NMTGAN_TRY(sum(p.part, p.slices, a->M, p.coef, (T*)dh, ld_dh));
  return 0;
}
static int xent_grads_16(const nmtgan_xent_args* a, const float* lse, const float* grad_row, void* dh, int64_t ld_dh, void* dw,
                         int64_t ld_dw, void* ws, size_t ws_bytes, hipStream_t st) {
  using T = bf16_t;
  XentPlan q;
  carve_xent(a, (char*)ws, ws_bytes, q);
  const float low = xent_low(a), high = 1.f - a->smoothing - low;
  const float unit = high != 0.f ? high : 1.f;
  XentPrep pr{};
  pr.h = a->h; pr.w = a->w; pr.ldh = a->ldh; pr.ldw = a->ldw;
  pr.labels = a->labels; pr.grad_row = grad_row; pr.lse = lse;
  pr.coef = q.coef; pr.factor = q.factor; pr.inv_unit = 1.f / unit; pr.lse2 = q.lse2; pr.label = q.label; pr.ht = q.ht; pr.part = q.colsum;
  pr.M = a->M; pr.Mp = q.rows_padded; pr.V = a->V; pr.d = a->d;
  pr.n_rows = (q.rows_padded + 255) / 256;
  pr.n_turn = q.rows_padded / 64 * ((a->d + 63) / 64);
  hipLaunchKernelGGL(xent_prep_kernel<T>, dim3(pr.n_rows + pr.n_turn + (low > 0.f ? SUM_W + SUM_H : 0)), dim3(256), 0, st, pr);
  NMTGAN_CHECK_LAUNCH("linear_xent_prep");
  if (low > 0.f) {
    hipLaunchKernelGGL(xent_sums_kernel, dim3((a->d + 63) / 64, 2), dim3(1024), 0, st, q.colsum, a->d, -low,
                       q.part_w ? -low : -low / unit, q.wsum, q.hsum);
    NMTGAN_CHECK_LAUNCH("linear_xent_sums");
  }
  XentEpilogue x{};
  x.factor = q.factor; x.lse2 = q.lse2; x.label = q.label; x.y = q.y;
  x.rows_padded = q.rows_padded;
  x.piece_padded = q.piece;
  x.high = high;
  int used = 0;
  for (int v0 = 0; v0 < a->V; v0 += q.piece, ++used) {
    const int n = std::min(q.piece, a->V - v0);
    x.first = v0;
    const T* w = (const T*)a->w + (int64_t)v0 * a->ldw;
    NMTGAN_TRY(launch_gemm_xent(a->dtype, true, w, a->ldw, n, a->h, a->ldh, a->M, a->d, nullptr, x, st));
    NMTGAN_TRY(launch_gemm_kmajor(a->dtype, q.y, q.rows_padded, q.piece, w, a->ldw, n, a->M, a->d, q.slices, q.kt_slice,
                                  q.part + (int64_t)(used % q.sets) * q.slices * a->M * a->d, used >= q.sets, st));
    if (q.part_w) {
      NMTGAN_TRY(launch_gemm_kslice(a->dtype, q.y, q.rows_padded, q.ht, q.rows_padded, n, a->d, q.row_slices, q.kt_rows, q.part_w, st));
      hipLaunchKernelGGL(xent_dh_kernel<T>, dim3((unsigned)(((int64_t)n * a->d / 4 + 255) / 256)), dim3(256), 0, st, q.part_w,
                         q.row_slices, n, a->d, nullptr, unit, q.hsum, (T*)dw + (int64_t)v0 * ld_dw, ld_dw);
      NMTGAN_CHECK_LAUNCH("linear_xent_dw");
      continue;
    }
    nmtgan_gemm_args b{};
    b.op_dtype = a->dtype;
    b.epilogue = NMTGAN_EPI_LINEAR;
    b.A = q.y; b.lda = q.rows_padded; b.Wt = q.ht; b.bias = q.hsum;
    b.M = n; b.N = a->d; b.K = q.rows_padded;
    b.n_seg = 1; b.out[0] = (T*)dw + (int64_t)v0 * ld_dw; b.ldo[0] = ld_dw; b.seg_scale[0] = unit;
    SplitKScope scope(q.splitk, SPLITK_BYTES);
    NMTGAN_TRY(launch_gemm(&b, st));
  }
  hipLaunchKernelGGL(xent_dh_kernel<T>, dim3((unsigned)(((int64_t)a->M * a->d / 4 + 255) / 256)), dim3(256), 0, st, q.part, q.sets * q.slices,
                     a->M, a->d, q.coef, unit, q.wsum, (T*)dh, ld_dh);
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
  NMTGAN_REQUIRE(a->M <= 1 << 22, "linear_xent_grads: more than 2^22 rows (a column of d(logits) would outgrow its piece)");
  const size_t need = linear_xent_workspace(a, true);
  NMTGAN_REQUIRE(need == 0 || (ws && ws_bytes >= need && (uintptr_t)ws % 256 == 0),
                 "linear_xent_grads: workspace of %zu bytes (256-byte aligned) needed, %zu given", need, ws_bytes);
  const int64_t width = (int64_t)a->d * es;
  NMTGAN_TRY(refuse_overlaps("linear_xent_grads",
                             {Region("dh", dh, a->M, ld_dh * es, width), Region("dw", dw, a->V, ld_dw * es, width),
                              Region("workspace", ws, (int64_t)need)},
                             {Region("h", a->h, a->M, a->ldh * es, width), Region("w", a->w, a->V, a->ldw * es, width),
                              Region("labels", a->labels, 4LL * a->M), Region("lse", lse, 4LL * a->M),
                              Region("grad_row", grad_row, 4LL * a->M)}));
  if (a->M == 0) {
    const dim3 grid((unsigned)(((int64_t)a->V * a->d + 255) / 256));
    if (a->dtype == NMTGAN_F32) hipLaunchKernelGGL(xent_zero_rows_kernel<float>, grid, dim3(256), 0, st, (float*)dw, ld_dw, a->V, a->d);
    else hipLaunchKernelGGL(xent_zero_rows_kernel<bf16_t>, grid, dim3(256), 0, st, (bf16_t*)dw, ld_dw, a->V, a->d);
    NMTGAN_CHECK_LAUNCH("linear_xent_zero");
    return 0;
  }
  if (!direct_grads(a)) return xent_grads_16(a, lse, grad_row, dh, ld_dh, dw, ld_dw, ws, ws_bytes, st);
  if (a->dtype == NMTGAN_BF16) return direct_grads_t<bf16_t>(a, lse, grad_row, dh, ld_dh, dw, ld_dw, ws, ws_bytes, st);
  return direct_grads_t<float>(a, lse, grad_row, dh, ld_dh, dw, ld_dw, ws, ws_bytes, st);
}

}  // namespace nmtgan
