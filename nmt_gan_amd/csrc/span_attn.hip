// Span attention: the form for single tokens, checks and launches (span_tiles.h has the formulas).
#include "regions.h"
#include "span_tiles.h"

namespace nmtgan {

// ------------------------------------------------------------------------------------------ single tokens
// One query row and one key head with its query heads per workgroup, `splits` workgroups along the span; waves and splits
// are joined at the end in a fixed order.  Vector form (one query head per key head, and fp32 with up to GT): a key row is
// read once, as 16-byte chunks by LPK neighbouring lanes, so a wave reads 64 / LPK keys per instruction and STEP_U such
// groups of K and of V are in flight while the previous ones are used; every lane group keeps a softmax of its own (no
// exchange inside the loop but the LPK-lane sum of a dot product).
// Bound by the rate at which K and V come; where heads share a key, by the arithmetic per key (hence the matrix form below).  One
// row over 256 keys, 8 heads: 5.5 us, a launch and two dependent loads.
constexpr int STEP_U = 4;

template <int LPK>
__device__ __forceinline__ float key_sum(float v) {          // over the lanes of one key
  v = dpp_add<0xB1>(v);
  v = dpp_add<0x4E>(v);
  if constexpr (LPK >= 8) v = dpp_add<0x141>(v);
  if constexpr (LPK >= 16) v = dpp_add<0x140>(v);
  if constexpr (LPK >= 32) v += __shfl_xor(v, 16, 64);
  return v;
}
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true)));
}
// over the lanes that hold the same chunk of different keys (rotations by 8 and 4 inside 16 lanes, then across)
template <int LPK>
__device__ __forceinline__ float chunk_sum(float v) {
  if constexpr (LPK <= 8) v = dpp_add<0x128>(v);
  if constexpr (LPK <= 4) v = dpp_add<0x124>(v);
  if constexpr (LPK <= 16) return groups4_sum(v);
  else return both_halves_sum(v);
}
template <int LPK>
__device__ __forceinline__ float chunk_max(float v) {
  if constexpr (LPK <= 8) v = dpp_max<0x128>(v);
  if constexpr (LPK <= 4) v = dpp_max<0x124>(v);
  if constexpr (LPK <= 16) return groups4_max(v);
  else return both_halves_max(v);
}
template <typename T>
__device__ __forceinline__ void unpack_chunk(const uint4& r, float (&f)[16 / (int)sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
    unpack8<T>(r, f);
  } else {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
}

// one wave joins the four waves' parts of a head and hands them on: to the split's part, or as the result
// (acc + w * stride = wave w's output of this head)
template <typename T, int DP, typename B>
__device__ __forceinline__ void step_finish(const SpanParams& p, const float* acc, int stride, const B& s_m, const B& s_l, int i,
                                            int h, int t, int z, int splits, float* part, float* xs, int lane) {
  const float mt = fmaxf(fmaxf(s_m[0][t], s_m[1][t]), fmaxf(s_m[2][t], s_m[3][t])), mu = mt == -INFINITY ? 0.f : mt;
  float r[4], lt = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    r[k] = __builtin_amdgcn_exp2f(s_m[k][t] - mu);
    lt += s_l[k][t] * r[k];
  }
  const int64_t at = (int64_t)i * p.heads + h;
  float* mine = part + (at * splits + z) * (p.dh + 2);
  float o[DP > 64 ? 2 : 1];
  bool fine = lt < INFINITY;
#pragma unroll
  for (int u = 0; u < (DP > 64 ? 2 : 1); ++u) {
    const int c = lane + 64 * u;
    o[u] = c < p.dh ? (acc[c] * r[0] + acc[stride + c] * r[1]) + (acc[2 * stride + c] * r[2] + acc[3 * stride + c] * r[3]) : 0.f;
    fine = fine && fmaf(o[u], 0.f, 0.f) == 0.f;
  }
  if (splits > 1) {
#pragma unroll
    for (int u = 0; u < (DP > 64 ? 2 : 1); ++u)
      if (lane + 64 * u < p.dh) mine[lane + 64 * u] = o[u];
    if (lane == 0) {
      mine[p.dh] = mt;
      mine[p.dh + 1] = lt;
    }
    return;
  }
  if (__any(!fine)) {                                        // (padding of a tile met an infinity): exactly, by itself
    span_fwd_row<T>(p, i, h, xs, lane);
    return;
  }
#pragma unroll
  for (int u = 0; u < (DP > 64 ? 2 : 1); ++u)
    if (lane + 64 * u < p.dh)
      OpTraits<T>::store((T*)p.out + (int64_t)i * p.ldo + h * p.dh + lane + 64 * u, lt == 0.f ? 0.f : o[u] / lt);
  if (p.lse && lane == 0) p.lse[at] = lt == 0.f ? -INFINITY : mt * LN2 + logf(lt);
}

template <typename T, int DP, int GT, int FORM>
__global__ __launch_bounds__(256) void span_step_kernel(SpanParams p, int splits, int groups, float* part) {
  constexpr int EPC = 16 / (int)sizeof(T), LPK = DP / EPC, KPW = 64 / LPK, KB = STEP_U * KPW;
  constexpr bool EXTRA = FORM != SPAN_PLAIN, LIBRARY = library_tanh<T, FORM>;
  __shared__ float s_acc[4][GT][DP];
  __shared__ float s_m[4][GT], s_l[4][GT], s_xs[4][SPAN_MAX_DH];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, dh = p.dh, g = p.heads / p.kv_heads;
  const int i = blockIdx.x / splits, z = blockIdx.x % splits;
  const int kvh = blockIdx.y / groups, h0 = kvh * g + (blockIdx.y % groups) * GT, ng = min(GT, (kvh + 1) * g - h0);
  const int c = (lane % LPK) * EPC, kk = lane / LPK;
  const int2 sp = span_of(p, i);
  const int64_t len = sp.y - sp.x;
  const int j0 = sp.x + (int)(len * z / splits), j1 = sp.x + (int)(len * (z + 1) / splits);
  const bool has = c < dh;
  const T* K = (const T*)p.k + kvh * dh + c;
  const T* V = (const T*)p.v + kvh * dh + c;
  const float f = EXTRA ? 1.f : p.scale * LOG2E;             // products come out in units of log 2
  float q[GT][EPC], acc[GT][EPC], m[GT], l[GT], slope[GT];
#pragma unroll
  for (int u = 0; u < GT; ++u) {
    uint4 r = make_uint4(0, 0, 0, 0);
    if (has && u < ng) r = *reinterpret_cast<const uint4*>((const T*)p.q + (int64_t)i * p.ldq + (h0 + u) * dh + c);
    unpack_chunk<T>(r, q[u]);
    m[u] = -INFINITY;
    l[u] = slope[u] = 0.f;
    if (EXTRA && p.slopes && u < ng) slope[u] = p.slopes[h0 + u] * LOG2E;
#pragma unroll
    for (int e = 0; e < EPC; ++e) {
      q[u][e] *= f;
      acc[u][e] = 0.f;
    }
  }
  const int pos = EXTRA ? pos_of(p, i) : 0;
  const float inv_cap = EXTRA && p.cap > 0.f ? p.scale / p.cap : 0.f, cap2 = p.cap * LOG2E;
  const bool few = __builtin_amdgcn_readfirstlane((int)len) <= SPAN_SHORT;      // see cap_scores_fine

  uint4 kr[STEP_U], vr[STEP_U];
  auto fetch = [&](int b) {
#pragma unroll
    for (int u = 0; u < STEP_U; ++u) {
      const int j = b + u * KPW + kk;
      const bool ok = has && j < j1;
      kr[u] = ok ? *reinterpret_cast<const uint4*>(K + (int64_t)j * p.ldk) : make_uint4(0, 0, 0, 0);
      vr[u] = ok ? *reinterpret_cast<const uint4*>(V + (int64_t)j * p.ldv) : make_uint4(0, 0, 0, 0);
    }
  };
  int b = j0 + KB * w;
  if (b < j1) fetch(b);
  for (; b < j1; b += 4 * KB) {
    uint4 ka[STEP_U], va[STEP_U];
#pragma unroll
    for (int u = 0; u < STEP_U; ++u) { ka[u] = kr[u]; va[u] = vr[u]; }
    if (b + 4 * KB < j1) fetch(b + 4 * KB);
    float s[STEP_U][GT];
#pragma unroll
    for (int u = 0; u < STEP_U; ++u) {
      float x[EPC];
      unpack_chunk<T>(ka[u], x);
      const int j = b + u * KPW + kk;
#pragma unroll
      for (int t = 0; t < GT; ++t) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < EPC; ++e) d = fmaf(x[e], q[t][e], d);
        d = key_sum<LPK>(d);
        if constexpr (EXTRA) {
          if (p.cap > 0.f) d = few ? cap_score<LIBRARY>(d * inv_cap, cap2, SMALL_TANH) : cap_score<LIBRARY>(d * inv_cap, cap2, 0.f);
          else d *= p.scale * LOG2E;
          if (p.slopes) d = fmaf(-slope[t], fabsf((float)(pos - j)), d);
        }
        s[u][t] = j < j1 ? d : -INFINITY;
      }
    }
#pragma unroll
    for (int t = 0; t < GT; ++t) {
      float mx = s[0][t];
#pragma unroll
      for (int u = 1; u < STEP_U; ++u) mx = fmaxf(mx, s[u][t]);
      const float mn = fmaxf(m[t], mx), mu = mn == -INFINITY ? 0.f : mn;
      if (__any(mn > m[t])) {
        const float r = __builtin_amdgcn_exp2f(m[t] - mu);
        l[t] *= r;
#pragma unroll
        for (int e = 0; e < EPC; ++e) acc[t][e] *= r;
        m[t] = mn;
      }
#pragma unroll
      for (int u = 0; u < STEP_U; ++u) {
        s[u][t] = __builtin_amdgcn_exp2f(s[u][t] - mu);
        l[t] += s[u][t];
      }
    }
#pragma unroll
    for (int u = 0; u < STEP_U; ++u) {
      float x[EPC];
      unpack_chunk<T>(va[u], x);
#pragma unroll
      for (int t = 0; t < GT; ++t)
#pragma unroll
        for (int e = 0; e < EPC; ++e) acc[t][e] = fmaf(s[u][t], x[e], acc[t][e]);
    }
  }
#pragma unroll
  for (int t = 0; t < GT; ++t) {
    const float mt = chunk_max<LPK>(m[t]), mu = mt == -INFINITY ? 0.f : mt, r = __builtin_amdgcn_exp2f(m[t] - mu);
    const float lt = chunk_sum<LPK>(l[t] * r);
#pragma unroll
    for (int e = 0; e < EPC; ++e) {
      const float a = chunk_sum<LPK>(acc[t][e] * r);
      if (kk == 0) s_acc[w][t][c + e] = a;
    }
    if (lane == 0) { s_m[w][t] = mt; s_l[w][t] = lt; }
  }
  __syncthreads();
  for (int t = w; t < ng; t += 4) step_finish<T, DP>(p, s_acc[0][t], GT * DP, s_m, s_l, i, h0 + t, t, z, splits, part, s_xs[w], lane);
}

// The same with the matrix cores, 16-bit types and 2 to 16 query heads per key head: the heads are the 16 columns of 16x16
// products over tiles of 32 keys (S^T = K Q^T, out^T = V^T P^T, layouts as in span_tiles.h with four lanes a softmax row),
// so the work per key does not grow with the heads.  Each wave walks every fourth tile of its split through LDS of its own.
// 48 rows over 522499 keys together (up to 16384 each), 8 heads of 64 over 2, capped, fp16: 53 us = 5.07 TB/s, the rate of a
// large copy here; the vector form took 82 us.
typedef float f32x4_t __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ f32x4_t mma16x16(const uint4& a, const uint4& b, f32x4_t c) {
  if constexpr (__is_same(T, bf16_t)) {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
}
template <typename T, int DP, int FORM>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void span_step_heads_kernel(SpanParams p, int splits, int groups, float* part) {
  using G = Geo<T, DP>;
  using D = Dma<T, DP>;
  constexpr bool EXTRA = FORM != SPAN_PLAIN, LIBRARY = library_tanh<T, FORM>;
  constexpr int NS = DP <= 64 ? 3 : 2, STAGE = 2 * D::BYTES, KS = DP / 32, DB = DP / 16;      // stages, k-steps, dh blocks
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ float s_m[4][16], s_l[4][16], xs[4][SPAN_MAX_DH];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int dh = p.dh, g = p.heads / p.kv_heads, col = lane & 15, q4 = lane >> 4;
  const int i = blockIdx.x / splits, z = blockIdx.x % splits;
  const int kvh = blockIdx.y / groups, h0 = kvh * g + (blockIdx.y % groups) * 16, ng = min(16, (kvh + 1) * g - h0);
  int2 sp = span_of(p, i);
  sp.x = __builtin_amdgcn_readfirstlane(sp.x);
  sp.y = __builtin_amdgcn_readfirstlane(sp.y);
  const int64_t len = sp.y - sp.x;
  const int j0 = sp.x + (int)(len * z / splits), j1 = sp.x + (int)(len * (z + 1) / splits);
  const T* K = (const T*)p.k + kvh * dh;
  const T* V = (const T*)p.v + kvh * dh;
  unsigned char* mine = smem + w * NS * STAGE;
  const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) void*)mine);
  D dk, dv;
  dk.init(p.ldk, dh, lane);
  dv.init(p.ldv, dh, lane);
  const int nt = (j1 - j0 + 31) / 32;
  auto issue = [&](int t, int buf) {
    dk.issue(K, p.ldk, j0 + 32 * t, j1 - j0 - 32 * t, lds + buf * STAGE, lane);
    dv.issue(V, p.ldv, j0 + 32 * t, j1 - j0 - 32 * t, lds + buf * STAGE + D::BYTES, lane);
  };
#pragma unroll
  for (int k = 0; k < NS; ++k)
    if (w + 4 * k < nt) issue(w + 4 * k, k);
  uint4 own[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    const int c = 32 * k + 8 * q4;
    own[k] = col < ng && c < dh ? *reinterpret_cast<const uint4*>((const T*)p.q + (int64_t)i * p.ldq + (h0 + col) * dh + c)
                                : make_uint4(0, 0, 0, 0);
  }
  const float sc2 = p.scale * LOG2E;
  const float slope2 = EXTRA && p.slopes && col < ng ? p.slopes[h0 + col] * LOG2E : 0.f;
  const int pos = EXTRA ? pos_of(p, i) : 0;
  const float cap2 = p.cap * LOG2E, inv_cap = p.cap > 0.f ? p.scale / p.cap : 0.f;
  const float inv2 = inv_cap * 2.f * LOG2E;
  const bool fine = LIBRARY || (int)len <= SPAN_SHORT;       // see cap_scores_fine
  f32x4_t acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  int buf = 0;
  for (int t = w; t < nt; t += 4) {
    if (NS == 3 && t + 8 < nt) wait_dma<4 * D::NI>();
    else if (t + 4 < nt) wait_dma<2 * D::NI>();
    else wait_dma<0>();
    const unsigned char* tk = mine + buf * STAGE;
    const unsigned char* tv = tk + D::BYTES;
    float s[8];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f32x4_t c = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k)
        c = mma16x16<T>(*reinterpret_cast<const uint4*>(tk + G::swz(16 * kb + col, 4 * k + q4)), own[k], c);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * kb + r] = c[r];
    }
    const int first = j0 + 32 * t + 4 * q4;                  // key of s[0]; s[4 kb + r] is key first + 16 kb + r
    if (EXTRA && p.cap > 0.f && !fine) {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        s[r] = fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[r] * inv2)), -2.f * cap2, cap2);
    } else if (EXTRA && p.cap > 0.f) {
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = cap_score<LIBRARY>(s[r] * inv_cap, cap2, SMALL_TANH);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] *= sc2;
    }
    if (EXTRA && p.slopes) {
      const float away = (float)(pos - first);
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = fmaf(-slope2, fabsf(away - (float)(16 * (r >> 2) + (r & 3))), s[r]);
    }
    if (j0 + 32 * t + 32 > j1) {
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = first + 16 * (r >> 2) + (r & 3) < j1 ? s[r] : -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    mx = groups4_max(mx);
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx), c = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
      l *= c;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[db][r] *= c;
      m = mn;
    }
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      s[r] = __builtin_amdgcn_exp2f(s[r] - mu);
      l += s[r];
    }
    const uint4 pb = make_uint4(pack_pair<T>(s[0], s[1]), pack_pair<T>(s[2], s[3]), pack_pair<T>(s[4], s[5]), pack_pair<T>(s[6], s[7]));
    const int row = 4 * q4 + (col >> 2);
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int c = 16 * db + 4 * (lane & 3);
      const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                     (lds_s16x4_p)(tv + G::swz(row, c >> 3) + 2 * (c & 7))));
      const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                     (lds_s16x4_p)(tv + G::swz(row + 16, c >> 3) + 2 * (c & 7))));
      acc[db] = mma16x16<T>(make_uint4(lo.x, lo.y, hi.x, hi.y), pb, acc[db]);
    }
    if (t + 4 * NS < nt) {
      wait_lds();
      issue(t + 4 * NS, buf);
    }
    buf = buf + 1 == NS ? 0 : buf + 1;
  }
  l = groups4_sum(l);
  if (lane < 16) { s_m[w][lane] = m; s_l[w][lane] = l; }
#pragma unroll
  for (int db = 0; db < DB; ++db)
    *reinterpret_cast<float4*>(mine + (col * DP + 16 * db + 4 * q4) * 4) = make_float4(acc[db][0], acc[db][1], acc[db][2], acc[db][3]);
  __syncthreads();
  const float* out = reinterpret_cast<const float*>(smem);
  for (int t = w; t < ng; t += 4) step_finish<T, DP>(p, out + t * DP, NS * STAGE / 4, s_m, s_l, i, h0 + t, t, z, splits, part, xs[w], lane);
}

// one wave per (row, head): the splits' parts, in order (48 rows x 8 heads x 11 parts: 4.8 us, a launch's latency)
template <typename T>
__global__ __launch_bounds__(256) void span_join_kernel(SpanParams p, int splits, const float* part) {
  __shared__ float xs[4][SPAN_MAX_DH];
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= (int64_t)p.M * p.heads) return;
  const int i = (int)(t / p.heads), h = (int)(t % p.heads), dh = p.dh;
  const float* o = part + t * splits * (dh + 2);
  // splits <= 64: lane z holds split z's maximum and sum
  const float mz = lane < splits ? o[lane * (dh + 2) + dh] : -INFINITY, lz = lane < splits ? o[lane * (dh + 2) + dh + 1] : 0.f;
  const float m = wave_max(mz), mu = m == -INFINITY ? 0.f : m, rz = __builtin_amdgcn_exp2f(mz - mu);
  const float l = wave_sum(lz * rz);
  float acc[2] = {0.f, 0.f};
  bool fine = l < INFINITY;
#pragma unroll
  for (int u = 0; u < 2; ++u) {                              // every lane stays in the loop: it answers the exchange
    if (64 * u >= dh) break;
    const int c = min(64 * u + lane, dh - 1);
    for (int z = 0; z < splits; z += 8) {                    // eight parts in flight
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = o[min(z + k, splits - 1) * (dh + 2) + c];
#pragma unroll
      for (int k = 0; k < 8; ++k) acc[u] = fmaf(z + k < splits ? v[k] : 0.f, __shfl(rz, min(z + k, 63), 64), acc[u]);
    }
    fine = fine && fmaf(acc[u], 0.f, 0.f) == 0.f;
  }
  if (__any(!fine)) {
    span_fwd_row<T>(p, i, h, xs[threadIdx.x >> 6], lane);
    return;
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (64 * u + lane < dh)
      OpTraits<T>::store((T*)p.out + (int64_t)i * p.ldo + h * dh + 64 * u + lane, l == 0.f ? 0.f : acc[u] / l);
  if (p.lse && lane == 0) p.lse[t] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
}

// ------------------------------------------------------------------------------------------ host
static bool rows_ok(const void* ptr, int64_t ld, int64_t width, int es) {
  return (uintptr_t)ptr % 16 == 0 && ld >= width && ld * es % 16 == 0;
}
static int fill_span(const nmtgan_span_args* a, SpanParams& p, const char* what) {
  NMTGAN_REQUIRE(a != nullptr, "%s: null args", what);
  NMTGAN_REQUIRE(valid_op_dtype(a->dtype), "%s: bad dtype %d", what, a->dtype);
  constexpr int MOST = INT32_MAX - 65536;         // indexes run over the end of the last tile
  NMTGAN_REQUIRE(a->M >= 0 && a->N >= 0 && a->M <= MOST && a->N <= MOST, "%s: bad shape M=%d N=%d", what, a->M, a->N);
  NMTGAN_REQUIRE(a->heads > 0 && a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->heads <= 4096,
                 "%s: heads=%d must be a multiple of kv_heads=%d, at most 4096", what, a->heads, a->kv_heads);
  NMTGAN_REQUIRE(a->dh > 0 && a->dh % 8 == 0 && a->dh <= SPAN_MAX_DH, "%s: head width %d must be a multiple of 8, at most %d",
                 what, a->dh, SPAN_MAX_DH);
  NMTGAN_REQUIRE(isfinite(a->scale) && isfinite(a->cap) && a->cap >= 0.f, "%s: scale and cap must be finite, cap >= 0", what);
  const int es = dtype_size(a->dtype);
  NMTGAN_REQUIRE(a->ldq < (1 << 24) && a->ldk < (1 << 24) && a->ldv < (1 << 24), "%s: rows further than 2^24 elements apart", what);
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

// what every form reads
static Region region(const char* name, const void* at, int64_t rows, int64_t ld, int64_t width, int es) {
  return Region(name, at, rows, ld * es, width * es);
}
#define SPAN_INPUTS(a, wq, wk, es)                                                                            \
  region("q", (a)->q, (a)->M, (a)->ldq, wq, es), region("k", (a)->k, (a)->N, (a)->ldk, wk, es),               \
      region("v", (a)->v, (a)->N, (a)->ldv, wk, es), Region("lo", (a)->lo, 4LL * (a)->M),                     \
      Region("hi", (a)->hi, 4LL * (a)->M), Region("pos", (a)->pos, 4LL * (a)->M), Region("slopes", (a)->slopes, 4LL * (a)->heads)
// of the forward forms
static int span_overlaps(const nmtgan_span_args* a, const void* ws, size_t ws_bytes, const char* what) {
  const int es = dtype_size(a->dtype);
  const int64_t wq = (int64_t)a->heads * a->dh, wk = (int64_t)a->kv_heads * a->dh;
  return refuse_overlaps(what, {region("out", a->out, a->M, a->ldo, wq, es), Region("lse", a->lse, 4LL * a->M * a->heads),
                                Region("workspace", ws, (int64_t)ws_bytes)},
                         {SPAN_INPUTS(a, wq, wk, es)});
}

int launch_attn_span(const nmtgan_span_args* a, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  SpanParams p;
  NMTGAN_TRY(fill_span(a, p, "attn_span"));
  if (p.M == 0) return 0;
  NMTGAN_TRY(span_overlaps(a, nullptr, 0, "attn_span"));
  return span_fwd_tiles(a->dtype, p, st);
}

// Workgroups along a span: enough to fill the chip four workgroups deep, none with less than 512 keys, and none but one
// below 1024 keys - the second launch that joins them costs more than the walk.  max_keys is a hint (the cut is made of the
// true length on the device), so a wrong one costs time only.  No more than 64, a lane each in the joining wave: one request
// over 2^20 keys then reads at 5.4 TB/s with 8 key heads of 64, 3.5 with 2, and at 2.5 to 2.8 with one (64 or 128 wide), which
// leaves three of four CUs without work; four requests of 2^18 keys with one key head of 128: 5.1.
static int span_splits(int M, int kv_heads, int max_keys) {
  if (max_keys <= 1024) return 1;
  const int64_t groups = std::max<int64_t>(1, (int64_t)M * kv_heads);
  const int64_t fill = (1024 + groups - 1) / groups;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(fill, 64), (max_keys + 511) / 512));
}
size_t attn_span_step_workspace(int M, int heads, int kv_heads, int dh, int max_keys) {
  if (M <= 0 || heads <= 0 || kv_heads <= 0 || dh <= 0) return 0;
  const int splits = span_splits(M, kv_heads, max_keys);
  return splits == 1 ? 0 : (size_t)M * heads * splits * (dh + 2) * sizeof(float);
}
template <typename T, int DP, int GT>
static int launch_step(const SpanParams& p, int splits, float* part, hipStream_t st) {
  const int groups = (p.heads / p.kv_heads + GT - 1) / GT;
  const dim3 grid((unsigned)(p.M * splits), p.kv_heads * groups);
  return with_form<T>(p, [&](auto form) -> int {
    hipLaunchKernelGGL((span_step_kernel<T, DP, GT, decltype(form)::value>), grid, dim3(256), 0, st, p, splits, groups, part);
    NMTGAN_CHECK_LAUNCH("attn_span_step");
    return 0;
  });
}
template <typename T, int DP>
static int launch_step_heads(const SpanParams& p, int splits, float* part, hipStream_t st) {
  constexpr size_t smem = (size_t)4 * (DP <= 64 ? 3 : 2) * 2 * Dma<T, DP>::BYTES;
  const int groups = (p.heads / p.kv_heads + 15) / 16;
  const dim3 grid((unsigned)(p.M * splits), p.kv_heads * groups);
  return with_form<T>(p, [&](auto form) -> int {
    constexpr int FORM = decltype(form)::value;
    NMTGAN_TRY(raise_lds(&span_step_heads_kernel<T, DP, FORM>, smem, "attn_span_step"));
    hipLaunchKernelGGL((span_step_heads_kernel<T, DP, FORM>), grid, dim3(256), smem, st, p, splits, groups, part);
    NMTGAN_CHECK_LAUNCH("attn_span_step");
    return 0;
  });
}
template <typename T, int DP>
static int choose_step(const SpanParams& p, int splits, float* part, hipStream_t st) {
  const int g = p.heads / p.kv_heads;
  if (g == 1) return launch_step<T, DP, 1>(p, splits, part, st);
  if constexpr (sizeof(T) == 2) {
    return launch_step_heads<T, DP>(p, splits, part, st);
  } else {
    if (g == 2) return launch_step<T, DP, 2>(p, splits, part, st);
    if (g <= 4) return launch_step<T, DP, 4>(p, splits, part, st);
    return launch_step<T, DP, 8>(p, splits, part, st);
  }
}
int launch_attn_span_step(const nmtgan_span_args* a, int max_keys, void* ws, size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  SpanParams p;
  NMTGAN_TRY(fill_span(a, p, "attn_span_step"));
  NMTGAN_REQUIRE(max_keys >= 0, "attn_span_step: max_keys=%d", max_keys);
  if (p.M == 0) return 0;
  const size_t need = attn_span_step_workspace(p.M, p.heads, p.kv_heads, p.dh, max_keys);
  NMTGAN_REQUIRE(need == 0 || (ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0),
                 "attn_span_step: workspace of %zu bytes needed, %zu given", need, ws_bytes);
  const int splits = span_splits(p.M, p.kv_heads, max_keys);
  NMTGAN_REQUIRE((int64_t)p.M * splits < (1LL << 31) && ((int64_t)p.M * p.heads + 3) / 4 < (1LL << 31), "attn_span_step: too many rows");
  NMTGAN_TRY(span_overlaps(a, ws, need, "attn_span_step"));
  NMTGAN_DISPATCH_OP(a->dtype, T, {
    if (p.dh <= 32) NMTGAN_TRY((choose_step<T, 32>(p, splits, (float*)ws, st)));
    else if (p.dh <= 64) NMTGAN_TRY((choose_step<T, 64>(p, splits, (float*)ws, st)));
    else NMTGAN_TRY((choose_step<T, 128>(p, splits, (float*)ws, st)));
    if (splits == 1) return 0;
    hipLaunchKernelGGL(span_join_kernel<T>, dim3((unsigned)(((int64_t)p.M * p.heads + 3) / 4)), dim3(256), 0, st, p, splits,
                       (const float*)ws);
  });
  NMTGAN_CHECK_LAUNCH("attn_span_join");
  return 0;
}

static size_t carve_span_grads(int M, int heads, char* base, SpanParams* p) {
  const size_t nb = ((size_t)M + 31) / 32;
  const size_t a = align_up(nb * heads * 64 * sizeof(float), 256), b = align_up(nb * sizeof(int4), 256), c = align_up(nb * 64 * sizeof(int), 256);
  if (p) {
    p->rec = (float*)base;
    p->hull = (int4*)(base + a);
    p->spans = (int*)(base + a + b);
    p->posr = (int*)(base + a + b + c);
    p->chunk = (int2*)(base + a + b + 2 * c);
  }
  return a + b + 2 * c + (nb > LIST_STEP ? align_up((nb + LIST_STEP - 1) / LIST_STEP * sizeof(int2), 256) : 0);
}
size_t attn_span_grads_workspace(int M, int heads) { return M > 0 && heads > 0 ? carve_span_grads(M, heads, nullptr, nullptr) : 0; }
int launch_attn_span_grads(const nmtgan_span_args* a, const nmtgan_span_grads* g, void* ws, size_t ws_bytes, hipStream_t st) {
  prof::Scope prof_scope(prof::OTHER, st);
  SpanParams p;
  NMTGAN_TRY(fill_span(a, p, "attn_span_grads"));
  NMTGAN_REQUIRE(g != nullptr, "attn_span_grads: null gradients");
  NMTGAN_REQUIRE(a->dtype != NMTGAN_F16, "attn_span_grads: bf16 or fp32 (fp16 gradients would underflow without loss scaling)");
  const int es = dtype_size(a->dtype);
  NMTGAN_REQUIRE(g->ld_dout < (1 << 24), "attn_span_grads: rows further than 2^24 elements apart");
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
  NMTGAN_TRY(refuse_overlaps("attn_span_grads",
                             {region("dq", g->dq, p.M, g->ld_dq, wq, es), region("dk", g->dk, p.N, g->ld_dk, wk, es),
                              region("dv", g->dv, p.N, g->ld_dv, wk, es), Region("workspace", ws, (int64_t)need)},
                             {SPAN_INPUTS(a, wq, wk, es), region("out", a->out, p.M, a->ldo, wq, es),
                              region("dout", g->dout, p.M, g->ld_dout, wq, es), Region("lse", a->lse, 4LL * p.M * p.heads)}));
  if (p.M > 0) carve_span_grads(p.M, p.heads, (char*)ws, &p);
  p.dout = g->dout; p.ld_do = g->ld_dout; p.dq = g->dq; p.dk = g->dk; p.dv = g->dv;
  p.ld_dq = g->ld_dq; p.ld_dk = g->ld_dk; p.ld_dv = g->ld_dv;
  if (p.M > 0) {
    NMTGAN_TRY(span_dq_tiles(a->dtype, p, st));
  }
  return p.N > 0 ? span_dkv_tiles(a->dtype, p, st) : 0;
}

}  // namespace nmtgan
