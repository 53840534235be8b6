// Span attention: query row i attends to the keys lo[i] <= j < hi[i] of one packed key buffer.  Causal, document, prefix
// and padding masks of a packed (or padded) batch are all spans, so one kernel family serves teacher-forced training on
// packed sentences, prompts, and single tokens over a long cache.
//
//   r = scale q_i . k_j          t = tanh(r / cap), s = cap t   (s = r without a cap)
//   s -= slope_h |pos_i - j|     p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij)       out_i = sum_j p_ij v_j
//   dp = dout_i . v_j   delta_i = dout_i . out_i   dr = p (dp - delta_i) (1 - t^2) scale
//   dq_i = sum_j dr k_j    dk_j = sum_i dr q_i    dv_j = sum_i p dout_i   (sums over the heads that share a key head too)
//
// The tile kernels (span_fwd.hip, span_dq.hip, span_dkv.hip) multiply whole tiles on the matrix cores and give the pairs outside the
// spans the weight zero.  A NaN or an infinity in such a row would still come through (0 x NaN), so a wave that ends with
// a value that is not finite does those rows again with the row functions below: one row by one wave in plain fp32
// arithmetic over visible (row, key) pairs only.
#pragma once
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace nmtgan {

constexpr int SPAN_MAX_DH = 128;
constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.69314718055994531f;

struct SpanParams {
  const void* q; const void* k; const void* v;
  int64_t ldq, ldk, ldv, ldo;
  const int32_t* lo; const int32_t* hi; const int32_t* pos;
  const float* slopes;
  void* out; float* lse;
  int M, N, heads, kv_heads, dh;
  float scale, cap;
  int solo;                                      // a wave may walk a short span alone
  // gradients
  const void* dout; int64_t ld_do;
  void* dq; void* dk; void* dv;
  int64_t ld_dq, ld_dk, ld_dv;
  // per head and 32 rows: [lse / ln 2 x 32][delta x 32]; per 32 rows: [lo x 32][hi x 32] and [pos x 32][unused x 32]
  float* rec; int* spans; int* posr;
  int4* hull;                                    // [ceil(M / 32)] of 32 rows: keys seen by any row [x, y), by every row [z, w)
  int2* chunk;                                   // of LIST_STEP row blocks: keys seen by any; null where they are one chunk
};

__device__ __forceinline__ float span_exp(float x) { return __builtin_amdgcn_exp2f(x * LOG2E); }

// span of row i, cut to the key buffer; an empty one is (0, 0)
__device__ __forceinline__ int2 span_of(const SpanParams& p, int i) {
  const int a = max(p.lo[i], 0), b = min(p.hi[i], p.N);
  return b > a ? make_int2(a, b) : make_int2(0, 0);
}
__device__ __forceinline__ float* delta_at(const SpanParams& p, int i, int h) {
  return p.rec + (((int64_t)h * ((p.M + 31) / 32) + (i >> 5)) * 64 + 32 + (i & 31));
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
  const float lse = p.lse[(int64_t)i * p.heads + h], delta = *delta_at(p, i, h);
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
  const int nh = (p.M + 31) / 32;
  for (int b = 0; 2 * b < nh; ++b) {
    int4 hl = p.hull[2 * b];
    if (2 * b + 1 < nh) { const int4 o = p.hull[2 * b + 1]; hl = make_int4(min(hl.x, o.x), max(hl.y, o.y), 0, 0); }
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
                  *delta_at(p, i, h), p.slopes ? p.slopes[h] : 0.f, pos, j, pe, dr);
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

#define NMTGAN_DISPATCH_GRAD(dt, T, ...)                                          \
  do {                                                                            \
    if ((dt) == NMTGAN_BF16) { using T = ::nmtgan::bf16_t; __VA_ARGS__; }         \
    else { using T = float; __VA_ARGS__; }                                        \
  } while (0)

// ------------------------------------------------------------------------------------------ tiles on the matrix cores
// A wave owns 32 query rows (32 key rows in the dk/dv kernel) and walks the other side in tiles staged through LDS.
// Scores come transposed, S^T = K Q^T (32x32 products: lane & 31 = the wave's own row, 16 registers = rows of the tile), so
//   * a softmax row lives in the registers of two lanes (l, l ^ 32): its maximum and sum need one lane swap each;
//   * the same registers are the B operand of the second product (out^T = V^T P^T, dq^T = K^T dS^T, dv^T = dO^T P,
//     dk^T = Q^T dS) as they stand: which of a step's 16 tile rows sits in which k slot is free as long as A agrees, and A
//     is read in that order (ds_read_b64_tr_b16 turns 4 rows x 16 columns of the 16-bit tile; fp32 reads words).
// Rows of a tile are 16-byte chunks, XOR-swizzled so that 16 lanes that read one chunk of 16 rows hit 64 banks.
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_p;

template <typename T, int DP> struct Geo {
  static constexpr int RB = DP * (int)sizeof(T), CH = RB / 16, STEPS = RB / 32, DB = DP / 32;
  static constexpr int RPL = RB >= 256 ? 1 : 256 / RB, MASK = CH < 16 ? CH - 1 : 15;
  __device__ static __forceinline__ int swz(int row, int chunk) { return row * RB + ((chunk ^ ((row / RPL) & MASK)) << 4); }
};

template <typename T>
__device__ __forceinline__ f32x16_t mma_rows(const uint4& a, const uint4& b, f32x16_t c) {
  if constexpr (sizeof(T) == 2) {
    return mfma16<T>(a, b, c);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}
// s += tile rows [32 kb, +32) . own rows
template <typename T, int DP>
__device__ __forceinline__ f32x16_t score_block(const unsigned char* tile, int kb, const uint4 (&own)[Geo<T, DP>::STEPS], int lane) {
  using G = Geo<T, DP>;
  f32x16_t c;
#pragma unroll
  for (int r = 0; r < 16; ++r) c[r] = 0.f;
#pragma unroll
  for (int s = 0; s < G::STEPS; ++s) {
    const uint4 a = *reinterpret_cast<const uint4*>(tile + G::swz(32 * kb + (lane & 31), 2 * s + (lane >> 5)));
    c = mma_rows<T>(a, own[s], c);
  }
  return c;
}
template <typename T>
__device__ __forceinline__ unsigned pack_pair(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (__is_same(T, bf16_t)) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2{a, b}), b2));
  } else {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2{a, b}), f16x2_t));
  }
}
// A operand of 16 tile rows turned: rows row .. + 3 and row + 8 .. + 11 of 16 columns around `col`
template <typename T, int DP>
__device__ __forceinline__ uint4 turned_rows(const unsigned char* tile, int row, int col) {
  using G = Geo<T, DP>;
  const uint2 u = __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_p)(tile + G::swz(row, col >> 3) + 2 * (col & 7))));
  const uint2 v = __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_p)(tile + G::swz(row + 8, col >> 3) + 2 * (col & 7))));
  return make_uint4(u.x, u.y, v.x, v.y);
}
// acc^T[dh][own] += (tile^T)[dh][rows 32 kb ..] . x, x = a score block's registers
template <typename T, int DP>
__device__ __forceinline__ void accum_block(const unsigned char* tile, int kb, const f32x16_t& x, f32x16_t (&acc)[Geo<T, DP>::DB],
                                            int lane) {
  using G = Geo<T, DP>;
  const int hl = lane >> 5;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 b = make_uint4(pack_pair<T>(x[8 * t], x[8 * t + 1]), pack_pair<T>(x[8 * t + 2], x[8 * t + 3]),
                                 pack_pair<T>(x[8 * t + 4], x[8 * t + 5]), pack_pair<T>(x[8 * t + 6], x[8 * t + 7]));
      const int row = 32 * kb + 16 * t + 4 * hl + ((lane & 15) >> 2);
#pragma unroll
      for (int db = 0; db < G::DB; ++db)
        acc[db] = mfma16<T>(turned_rows<T, DP>(tile, row, 32 * db + (lane & 16) + 4 * (lane & 3)), b, acc[db]);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * kb + 8 * (r >> 2) + 4 * hl + (r & 3);
#pragma unroll
      for (int db = 0; db < G::DB; ++db) {
        const int col = 32 * db + (lane & 31);
        const float a = *reinterpret_cast<const float*>(tile + G::swz(row, col >> 2) + 4 * (col & 3));
        acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[r], acc[db], 0, 0, 0);
      }
    }
  }
}

// two accumulations over the same rows of a tile (16-bit types): the turned fragments serve both
template <typename T, int DP>
__device__ __forceinline__ void accum_two(const unsigned char* tile, const f32x16_t& x, const f32x16_t& y,
                                          f32x16_t (&accx)[Geo<T, DP>::DB], f32x16_t (&accy)[Geo<T, DP>::DB], int lane) {
  using G = Geo<T, DP>;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const uint4 bx = make_uint4(pack_pair<T>(x[8 * t], x[8 * t + 1]), pack_pair<T>(x[8 * t + 2], x[8 * t + 3]),
                                pack_pair<T>(x[8 * t + 4], x[8 * t + 5]), pack_pair<T>(x[8 * t + 6], x[8 * t + 7]));
    const uint4 by = make_uint4(pack_pair<T>(y[8 * t], y[8 * t + 1]), pack_pair<T>(y[8 * t + 2], y[8 * t + 3]),
                                pack_pair<T>(y[8 * t + 4], y[8 * t + 5]), pack_pair<T>(y[8 * t + 6], y[8 * t + 7]));
    const int row = 16 * t + 4 * (lane >> 5) + ((lane & 15) >> 2);
#pragma unroll
    for (int db = 0; db < G::DB; ++db) {
      const uint4 a = turned_rows<T, DP>(tile, row, 32 * db + (lane & 16) + 4 * (lane & 3));
      accx[db] = mfma16<T>(a, bx, accx[db]);
      accy[db] = mfma16<T>(a, by, accy[db]);
    }
  }
}
// own row as the B operand of score_block
template <typename T, int DP>
__device__ __forceinline__ void load_own(const T* row, bool ok, int dh, int lane, uint4 (&own)[Geo<T, DP>::STEPS]) {
#pragma unroll
  for (int s = 0; s < Geo<T, DP>::STEPS; ++s) {
    const int c = (2 * s + (lane >> 5)) * (16 / (int)sizeof(T));
    own[s] = ok && c < dh ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
  }
}
template <typename T>
__device__ __forceinline__ float chunk_dot(const uint4& a, const uint4& b) {
  float s = 0.f;
  if constexpr (sizeof(T) == 2) {
    float x[8], y[8];
    unpack8<T>(a, x);
    unpack8<T>(b, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(x[e], y[e], s);
  } else {
    s = __uint_as_float(a.x) * __uint_as_float(b.x);
    s = fmaf(__uint_as_float(a.y), __uint_as_float(b.y), s);
    s = fmaf(__uint_as_float(a.z), __uint_as_float(b.z), s);
    s = fmaf(__uint_as_float(a.w), __uint_as_float(b.w), s);
  }
  return s;
}
// transposed accumulators of the wave's own rows -> memory
template <typename T, int DP>
__device__ __forceinline__ void store_own(T* row, const f32x16_t (&acc)[Geo<T, DP>::DB], float f, int dh, int lane) {
#pragma unroll
  for (int db = 0; db < Geo<T, DP>::DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * db + 8 * g + 4 * (lane >> 5);
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[db][4 * g + e] * f;
      if (col < dh) VecIO<T, 4>::store(row + col, x);
    }
}
template <int DB>
__device__ __forceinline__ bool all_finite(const f32x16_t (&acc)[DB]) {
  float z = 0.f;                                  // x * 0 is 0 for every finite x and NaN for the others
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) z = fmaf(acc[db][r], 0.f, z);
  return z == 0.f;
}
template <int DB>
__device__ __forceinline__ void clear(f32x16_t (&acc)[DB]) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
}
__device__ __forceinline__ float both_halves_max(float v) {
  const u32x2_t b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float both_halves_sum(float v) {
  const u32x2_t b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What a launch's scores need.  EXTRA: a cap, a distance bias or the scale zero.  WIDE_CAP: with a cap above SPAN_WIDE, the 16-bit
// types only: tanh as 1 - 2 / (1 + exp(2 x)) is off by 2^-23 to 2^-22 absolute, a score by cap times that - up to 2^-16 at 64,
// far below the rounding of a probability to 16 bits, but 2^-3 at a cap of a million.  There, and in fp32, it is the library's tanh.
enum SpanForm { SPAN_PLAIN, SPAN_EXTRA, SPAN_WIDE_CAP };
constexpr float SPAN_WIDE = 64.f;
template <typename T, int FORM> constexpr bool library_tanh = sizeof(T) == 4 || FORM == SPAN_WIDE_CAP;
// tanh x = x - x^3/3 + 2 x^5/15 - 17 x^7/315 + 62 x^9/2835 - ..., below 1/4
__device__ __forceinline__ float small_tanh(float x) {
  const float y = x * x;
  return x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 62.f / 2835, -17.f / 315), 2.f / 15), -1.f / 3), 1.f);
}
constexpr float SMALL_TANH = 0.25f;
// cap tanh x in units of log 2 (c2 = cap / ln 2).  By the series where |x| < border, SMALL_TANH or 0
template <bool LIBRARY>
__device__ __forceinline__ float cap_score(float x, float c2, float border) {
  if constexpr (LIBRARY) return c2 * tanhf(x);
  const float d = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * (2.f * LOG2E)));
  return fabsf(x) < border ? c2 * small_tanh(x) : fmaf(d, -2.f * c2, c2);
}

struct WaveSpan { int lo, hi, all_lo, all_hi; };   // hull of a wave's spans; keys all of its rows see
template <int CTRL, bool MAX>
__device__ __forceinline__ int dpp_minmax(int v) {
  const int o = __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false);
  return MAX ? max(v, o) : min(v, o);
}
template <bool MAX>
__device__ __forceinline__ int rows_minmax(int v) { // over 32 lanes (both halves hold the same rows)
  v = dpp_minmax<0xB1, MAX>(v);
  v = dpp_minmax<0x4E, MAX>(v);
  v = dpp_minmax<0x141, MAX>(v);
  v = dpp_minmax<0x140, MAX>(v);
  const u32x2_t a = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  return __builtin_amdgcn_readfirstlane(MAX ? max((int)a[0], (int)a[1]) : min((int)a[0], (int)a[1]));
}
__device__ __forceinline__ WaveSpan wave_span(int2 sp) {
  return WaveSpan{rows_minmax<false>(sp.y > sp.x ? sp.x : 0x7fffffff), rows_minmax<true>(sp.y), rows_minmax<true>(sp.x),
                  rows_minmax<false>(sp.y)};
}
constexpr int SPAN_SHORT = 256;
// whether the spans of none of KW consecutive blocks of 32 rows reach over more than SPAN_SHORT keys
template <int KW>
__device__ __forceinline__ bool group_is_short(const SpanParams& p, int first, int* hull, int w, int lane) {
  const int i = (first + w) * 32 + (lane & 31);
  const WaveSpan ws = wave_span(i < p.M ? span_of(p, i) : make_int2(0, 0));
  if (lane == 0) hull[w] = ws.hi > ws.lo ? ws.hi - ws.lo : 0;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int k = 0; k < KW; ++k) n = max(n, hull[k]);
  return __builtin_amdgcn_readfirstlane(n) <= SPAN_SHORT;
}

// ------------------------------------------------------------------------------------------ split form
// The KW waves of a workgroup share their own 32 rows and take every KW-th 32-row tile of the other side, each into LDS of
// its own by DMA ahead of its use - no barrier inside the walk - and are joined at the end (against four row blocks per
// workgroup that share every tile: long documents 161 against 185 us forward when both existed).  Where a launch has
// workgroups enough without that (more than SPAN_FEW blocks of 32 rows times heads) and the spans of KW neighbouring blocks
// are short, one workgroup takes all KW, a wave each ("solo"), and the others leave: sentences of at most 50 tokens would
// give each of four waves less than a tile (32768 rows of them, forward: 39 us, 67 with four row blocks sharing tiles).
// Scalar base + one 32-bit lane offset per swizzle period; chunks behind dh and rows behind the last repeat a valid one
// (they meet zeros of the own rows or weights of zero).
// a pointer / offset that is the same in every lane, in scalar registers
__device__ __forceinline__ const char* scalar_ptr(const void* p) {
  const uint64_t a = (uint64_t)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)a), hi = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
  return (const char*)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ void dma16(unsigned voff, const void* sbase, unsigned lds_dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(voff), "s"(sbase), "s"(lds_dst)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(unsigned voff, const void* base, unsigned dst) {
  const char* sbase = scalar_ptr(base);
  const unsigned lds_dst = __builtin_amdgcn_readfirstlane(dst);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               :
               : "v"(voff), "s"(sbase), "s"(lds_dst)
               : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_dma() {       // at most N newer transfers may be in flight
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <typename T, int DP> struct Dma {
  using G = Geo<T, DP>;
  static constexpr int RPI = 64 / G::CH, NI = 32 / RPI;      // rows per instruction, instructions per 32 rows
  static constexpr int PERIOD = (G::MASK + 1) * G::RPL / RPI, NV = PERIOD < 1 ? 1 : PERIOD;
  static constexpr int BYTES = 32 * G::RB;
  unsigned off[NV];                                // lane's row inside an instruction and its chunk
  unsigned ldb;
  __device__ __forceinline__ void init(int64_t ld, int dh, int lane) {
    ldb = (unsigned)(ld * (int64_t)sizeof(T));
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int row = v * RPI + lane / G::CH, c = (lane % G::CH) ^ ((row / G::RPL) & G::MASK);
      off[v] = (unsigned)(lane / G::CH) * ldb + 16u * (unsigned)min(c, dh * (int)sizeof(T) / 16 - 1);
    }
  }
  // rows row0 .. row0 + 31 of `base`, row0 + left the first that is not there (left >= 1)
  __device__ __forceinline__ void issue(const T* base, int64_t ld, int row0, int left, unsigned dst, int lane) const {
    const char* b = scalar_ptr(reinterpret_cast<const char*>(base) + (int64_t)row0 * ld * (int64_t)sizeof(T));
    dst = __builtin_amdgcn_readfirstlane(dst);
    const unsigned step = __builtin_amdgcn_readfirstlane(ldb);
    const unsigned own = (unsigned)(lane / G::CH);
    if (left >= 32) {
#pragma unroll
      for (int u = 0; u < NI; ++u) dma16(off[u % NV], b + (uint64_t)(u * RPI) * step, dst + u * 1024);
    } else {
#pragma unroll
      for (int u = 0; u < NI; ++u) dma16(off[u % NV] + (min(own + u * RPI, (unsigned)left - 1u) - own) * ldb, b, dst + u * 1024);
    }
  }
};

// The tanh of a score block in place, in units of log 2: s = raw products -> capped scores minus `base`; BACK: t carries
// what (1 - t^2) is made of, see turned() - t itself from the library, else t = 1 - 2 d with d = 1 / (1 + exp(2 r / cap)), whose
// 1 - t^2 = 4 d (1 - d) leaves its 4 to the scale of the result
template <bool LIBRARY, bool BACK>
__device__ __forceinline__ void cap_scores(f32x16_t& s, f32x16_t& t, float scale, float cap, float base) {
  const float c2 = cap * LOG2E;
  if constexpr (LIBRARY) {
    const float inv = scale / cap;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float v = tanhf(s[r] * inv);
      s[r] = fmaf(c2, v, -base);
      if constexpr (BACK) t[r] = v;
    }
  } else {
    const float a = scale / cap * 2.f * LOG2E, c4 = -2.f * c2, c0 = c2 - base;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float d = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[r] * a));
      s[r] = fmaf(d, c4, c0);
      if constexpr (BACK) t[r] = d;
    }
  }
}
// The same of the 16-bit types, forward, where a row of the wave sees few keys (`fine`: this lane's does): the exponential's
// error, cap 2^-23 or more absolute, shows in the lse of a few small scores, so those rows take the series for them.  It goes by
// the row, not by its block: what a row is packed beside changes nothing in its scores.  Relative error of a score 2^-22 in the series,
// up to 2^-20 in the exponential's form, just above 1/4.  (8192 rows of documents up to 3626 long, capped at 30: 1 % of the forward pass.)
__device__ __forceinline__ void cap_scores_fine(f32x16_t& s, float scale, float cap, bool fine) {
  const float inv = scale / cap, c2 = cap * LOG2E, a = scale / cap * 2.f * LOG2E;
  const float border = fine ? SMALL_TANH : 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float x = s[r] * inv, d = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[r] * a));
    s[r] = fabsf(x) < border ? c2 * small_tanh(x) : fmaf(d, -2.f * c2, c2);
    if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);       // (not all sixteen at once: registers)
  }
}
template <bool LIBRARY>
__device__ __forceinline__ float turned(float t) { return LIBRARY ? fmaf(-t, t, 1.f) : fmaf(-t, t, t); }
template <bool LIBRARY>
__device__ __forceinline__ float result_scale(const SpanParams& p) { return p.cap > 0.f && !LIBRARY ? 4.f * p.scale : p.scale; }

// sums the KW waves' transposed accumulators (32 own rows x DP, each wave's in LDS at region w) and hands the result to
// put(row, col, x[4]) in whole rows; bad[row] is set where a sum is not finite
template <int DP> __device__ __forceinline__ int join_at(int row, int c4) { return row * DP + ((c4 ^ (row & (DP / 4 - 1))) << 2); }
template <int DP>
__device__ __forceinline__ void join_write(float* region, const f32x16_t (&acc)[DP / 32], float f, int lane) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c4 = 8 * db + 2 * g + (lane >> 5);
      *reinterpret_cast<float4*>(region + join_at<DP>(lane & 31, c4)) =
          make_float4(acc[db][4 * g] * f, acc[db][4 * g + 1] * f, acc[db][4 * g + 2] * f, acc[db][4 * g + 3] * f);
    }
}
template <int DP, int KW>
__device__ __forceinline__ float4 join_read(const float* region, int stride, int row, int c4) {
  float4 s = *reinterpret_cast<const float4*>(region + join_at<DP>(row, c4));
#pragma unroll
  for (int k = 1; k < KW; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(region + k * stride + join_at<DP>(row, c4));
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  return s;
}
__device__ __forceinline__ bool finite4(const float4& v) {
  return fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, v.w * 0.f))) == 0.f;
}

// dynamic LDS beyond 64 KiB has to be asked for once per device and kernel
template <typename F>
static inline int raise_lds(F* kernel, size_t bytes, const char* what) {
  if (bytes <= 48 * 1024) return 0;             // (the static part comes on top)
  NMTGAN_REQUIRE(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) ==
                     hipSuccess, "%s: cannot raise the dynamic LDS limit", what);
  return 0;
}
// f(form of these scores as a constant)
template <typename T, typename F>
static inline int with_form(const SpanParams& p, F f) {
  if constexpr (sizeof(T) == 2)
    if (p.cap > SPAN_WIDE) return f(std::integral_constant<int, SPAN_WIDE_CAP>{});
  if (p.cap > 0.f || p.slopes || p.scale == 0.f) return f(std::integral_constant<int, SPAN_EXTRA>{});
  return f(std::integral_constant<int, SPAN_PLAIN>{});
}
// Blocks of 32 rows (times heads) from which waves may walk alone: two workgroups of four waves on every SIMD.  Below it the
// chip is not full either way, and four waves a block finish sooner.
constexpr int64_t SPAN_FEW = 2048;
// Row blocks whose hulls the dk/dv kernel looks through at a time
constexpr int LIST_STEP = 1024;

int span_fwd_tiles(int dtype, const SpanParams& p, hipStream_t st);
int span_dq_tiles(int dtype, const SpanParams& p, hipStream_t st);
int span_dkv_tiles(int dtype, const SpanParams& p, hipStream_t st);

}  // namespace nmtgan
