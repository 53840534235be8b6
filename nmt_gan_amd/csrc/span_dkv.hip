// Span attention, gradients of keys and values on tiles (span_tiles.h has the formulas and the layout).
#include "span_tiles.h"

namespace nmtgan {

// dk, dv: a wave owns 32 keys of one key head and walks the query rows that may see them, head by head of the group.
// The walk goes by a list of row tiles whose hull meets the workgroup's keys, made by the first wave SPAN_LIST at a time.
constexpr int SPAN_LIST = 512;
template <typename T, int DP, int QT, int NW, bool EXTRA>
__global__ __launch_bounds__(64 * NW) void span_dkv_kernel(SpanParams p) {
  using G = Geo<T, DP>;
  constexpr int TB = QT * G::RB, NT = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];          // Q[2], dO[2], row scratch
  __shared__ __attribute__((aligned(16))) float s_lse[2][QT], s_delta[2][QT];
  __shared__ __attribute__((aligned(16))) int s_lo[2][QT], s_hi[2][QT], s_pos[2][QT];
  __shared__ __attribute__((aligned(16))) int4 hulls[SPAN_LIST];
  __shared__ int list[SPAN_LIST], n_list[2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int kvh = blockIdx.x % p.kv_heads, g = p.heads / p.kv_heads;
  const int k0 = blockIdx.x / p.kv_heads * 32 * NW, k1 = min(k0 + 32 * NW, p.N);
  const int w0 = k0 + 32 * w, j = w0 + (lane & 31), jc = min(j, p.N - 1);
  const bool ok = j < p.N;
  uint4 kf[G::STEPS], vf[G::STEPS];
  load_own<T, DP>((const T*)p.k + (int64_t)jc * p.ldk + kvh * p.dh, ok, p.dh, lane, kf);
  load_own<T, DP>((const T*)p.v + (int64_t)jc * p.ldv + kvh * p.dh, ok, p.dh, lane, vf);
  const float sc2 = p.scale * LOG2E;
  const float inv_cap = EXTRA && p.cap > 0.f ? 1.f / p.cap : 0.f;
  f32x16_t ak[G::DB], av[G::DB];
  clear(ak);
  clear(av);
  const int nq = (p.M + QT - 1) / QT;
  constexpr int HB = QT / 32;                     // hull entries of 32 rows per tile
  auto hull_of = [&](int t) {
    int4 a = p.hull[t * HB];
    if constexpr (HB == 2) {
      if (t * HB + 1 < (p.M + 31) / 32) {
        const int4 b = p.hull[t * HB + 1];
        a = make_int4(min(a.x, b.x), max(a.y, b.y), max(a.z, b.z), min(a.w, b.w));
      }
    }
    return a;
  };

  Stage<T, DP, QT, NT> sq, sd;
  float r_lse = 0.f, r_delta = 0.f;
  int r_lo = 0, r_hi = 0, r_pos = 0;
  auto fetch = [&](int tile, int h) {             // a row tile of head h into registers
    sq.load((const T*)p.q + h * p.dh, p.ldq, tile * QT, p.M, p.dh, tid);
    sd.load((const T*)p.dout + h * p.dh, p.ld_do, tile * QT, p.M, p.dh, tid);
    if (tid < QT) {
      const int i = tile * QT + tid;
      r_lo = r_hi = 0;
      r_lse = r_delta = 0.f;
      if (i < p.M) {
        const int2 sp = span_of(p, i);
        r_lo = sp.x;
        r_hi = sp.y;
        r_lse = delta_at(p, i, h)[-32];
        r_delta = *delta_at(p, i, h);
        if (EXTRA && p.slopes) r_pos = pos_of(p, i);
      }
    }
  };
  auto put = [&](int buf) {
    sq.store(smem + buf * TB, tid);
    sd.store(smem + (2 + buf) * TB, tid);
    if (tid < QT) {
      s_lse[buf][tid] = r_lse;
      s_delta[buf][tid] = r_delta;
      s_lo[buf][tid] = r_lo;
      s_hi[buf][tid] = r_hi;
      if (EXTRA) s_pos[buf][tid] = r_pos;
    }
  };

  for (int next = 0; next < nq;) {
    __syncthreads();
    if (w == 0) {
      int n = 0, b = next;
      for (; b < nq && n + 64 <= SPAN_LIST; b += 64) {
        bool on = false;
        int4 hl;
        if (b + lane < nq) {
          hl = hull_of(b + lane);
          on = hl.x < k1 && hl.y > k0;
        }
        const unsigned long long mask = __ballot(on);
        if (on) {
          const int at = n + __popcll(mask & ((1ull << lane) - 1));
          list[at] = b + lane;
          hulls[at] = hl;
        }
        n += __popcll(mask);
      }
      if (lane == 0) { n_list[0] = n; n_list[1] = b; }
    }
    __syncthreads();
    const int n = n_list[0], total = n * g;
    next = n_list[1];
    if (total == 0) continue;
    fetch(list[0], kvh * g);
    put(0);
    __syncthreads();
    for (int it = 0; it < total; ++it) {
      const int h = kvh * g + it / n, buf = it & 1;
      if (it + 1 < total) fetch(list[(it + 1) % n], kvh * g + (it + 1) / n);
      const int4 hl = hulls[it % n];
      if (hl.x < w0 + 32 && hl.y > w0) {
        const bool whole = hl.z <= w0 && hl.w >= w0 + 32 && w0 + 32 <= p.N;
        const unsigned char* tq = smem + buf * TB;
        const unsigned char* td = smem + (2 + buf) * TB;
        const float slope = EXTRA && p.slopes ? p.slopes[h] : 0.f;
#pragma unroll
        for (int qb = 0; qb < QT / 32; ++qb) {
          f32x16_t s = score_block<T, DP>(tq, qb, kf, lane);
          f32x16_t d = score_block<T, DP>(td, qb, vf, lane);
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const int row = 32 * qb + 8 * q4 + 4 * (lane >> 5);
            const float4 lse4 = *reinterpret_cast<const float4*>(&s_lse[buf][row]);
            const float4 del4 = *reinterpret_cast<const float4*>(&s_delta[buf][row]);
            int4 lo4 = make_int4(0, 0, 0, 0), hi4 = lo4, pos4 = lo4;
            if (!whole) {
              lo4 = *reinterpret_cast<const int4*>(&s_lo[buf][row]);
              hi4 = *reinterpret_cast<const int4*>(&s_hi[buf][row]);
            }
            if constexpr (EXTRA) pos4 = *reinterpret_cast<const int4*>(&s_pos[buf][row]);
            const float ls[4] = {lse4.x, lse4.y, lse4.z, lse4.w}, de[4] = {del4.x, del4.y, del4.z, del4.w};
            const int lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
            const int ps[4] = {pos4.x, pos4.y, pos4.z, pos4.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 4 * q4 + e;
              float turn = 1.f, x;
              if constexpr (EXTRA) x = score2<T>(p, s[r], inv_cap, slope, ps[e], j, turn) - ls[e];
              else x = fmaf(s[r], sc2, -ls[e]);
              float pe = __builtin_amdgcn_exp2f(x), ds = pe * (d[r] - de[e]);
              if constexpr (EXTRA) ds *= turn;
              if (!whole) {
                const bool on = (unsigned)(j - lo[e]) < (unsigned)(hi[e] - lo[e]);
                pe = on ? pe : 0.f;
                ds = on ? ds : 0.f;
              }
              s[r] = pe;
              d[r] = ds;
            }
          }
          accum_block<T, DP>(td, qb, s, av, lane);
          accum_block<T, DP>(tq, qb, d, ak, lane);
        }
      }
      if (it + 1 < total) put(buf ^ 1);
      __syncthreads();
    }
  }
  const unsigned long long bad = __ballot(ok && !(all_finite(ak) && all_finite(av)));
  if (ok && !((bad >> (lane & 31) | bad >> ((lane & 31) + 32)) & 1)) {
    store_own<T, DP>((T*)p.dk + (int64_t)j * p.ld_dk + kvh * p.dh, ak, p.scale, p.dh, lane);
    store_own<T, DP>((T*)p.dv + (int64_t)j * p.ld_dv + kvh * p.dh, av, 1.f, p.dh, lane);
  }
  if (bad) {
    float* x = reinterpret_cast<float*>(smem + 4 * TB) + w * 2 * SPAN_MAX_DH;
    for (unsigned left = (unsigned)bad | (unsigned)(bad >> 32); left; left &= left - 1)
      span_dkv_key<T>(p, w0 + __builtin_ctz(left), kvh, x, x + SPAN_MAX_DH, lane);
  }
}

// (128 list entries: two workgroups of head width 64 share a CU's LDS)
constexpr int SPLIT_LIST = 128;
template <typename T, int DP, int KW, bool EXTRA>
__global__ __launch_bounds__(64 * KW, DP * sizeof(T) <= 128 ? 2 : 1) void span_dkv_split_kernel(SpanParams p) {
  using G = Geo<T, DP>;
  using D = Dma<T, DP>;
  constexpr int STAGE = 2 * D::BYTES + 1024;      // Q, dO and the records of 32 rows
  constexpr int REGION = 2 * STAGE, NT = 64 * KW, JN = 32 * DP / 4 / NT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ __attribute__((aligned(16))) int4 hulls[SPLIT_LIST];
  __shared__ int list[SPLIT_LIST], n_list[2], bad[32];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % p.kv_heads, g = p.heads / p.kv_heads;
  const int k0 = blockIdx.x / p.kv_heads * 32, j = k0 + (lane & 31), jc = min(j, p.N - 1);
  const bool ok = j < p.N;
  unsigned char* mine = smem + w * REGION;
  const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) void*)mine);
  D dq, dd;
  dq.init(p.ldq, p.dh, lane);
  dd.init(p.ld_do, p.dh, lane);
  uint4 kf[G::STEPS], vf[G::STEPS];
  load_own<T, DP>((const T*)p.k + (int64_t)jc * p.ldk + kvh * p.dh, ok, p.dh, lane, kf);
  load_own<T, DP>((const T*)p.v + (int64_t)jc * p.ldv + kvh * p.dh, ok, p.dh, lane, vf);
  const float sc2 = p.scale * LOG2E;
  f32x16_t ak[G::DB], av[G::DB];
  clear(ak);
  clear(av);
  const int nb = (p.M + 31) / 32;
  const bool posr = EXTRA && p.slopes;
  constexpr int ND = 2 * D::NI + 2 + (EXTRA ? 1 : 0);        // transfers per tile (a record is one)
  auto issue = [&](int b, int h, int buf) {
    const unsigned dst = lds + buf * STAGE;
    dq.issue((const T*)p.q + h * p.dh, p.ldq, b * 32, p.M - b * 32, dst, lane);
    dd.issue((const T*)p.dout + h * p.dh, p.ld_do, b * 32, p.M - b * 32, dst + D::BYTES, lane);
    dma4(lane * 4, p.rec + ((int64_t)h * nb + b) * 64, dst + 2 * D::BYTES);
    dma4(lane * 4, p.spans + (int64_t)b * 64, dst + 2 * D::BYTES + 256);
    if constexpr (EXTRA) dma4(lane * 4, (posr ? p.posr : p.spans) + (int64_t)b * 64, dst + 2 * D::BYTES + 512);
  };

  for (int next = 0; next < nb;) {
    __syncthreads();
    if (w == 0) {
      int n = 0, b = next;
      for (; b < nb && n + 64 <= SPLIT_LIST; b += 64) {
        bool on = false;
        int4 hl;
        if (b + lane < nb) {
          hl = p.hull[b + lane];
          on = hl.x < k0 + 32 && hl.y > k0;
        }
        const unsigned long long mask = __ballot(on);
        if (on) {
          const int at = n + __popcll(mask & ((1ull << lane) - 1));
          list[at] = b + lane;
          hulls[at] = hl;
        }
        n += __popcll(mask);
      }
      if (lane == 0) { n_list[0] = n; n_list[1] = b; }
    }
    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(n_list[0]), total = n * g;
    next = __builtin_amdgcn_readfirstlane(n_list[1]);
    auto issue_nth = [&](int it, int buf) {
      issue(__builtin_amdgcn_readfirstlane(list[it % n]), kvh * g + it / n, buf);
    };
    if (w < total) issue_nth(w, 0);
    if (w + KW < total) issue_nth(w + KW, 1);
    int buf = 0;
    for (int it = w; it < total; it += KW, buf ^= 1) {
      const int h = kvh * g + it / n;
      const int4 hl = hulls[it % n];
      if (it + KW < total) wait_dma<ND>();
      else wait_dma<0>();
      const unsigned char* tq = mine + buf * STAGE;
      const unsigned char* td = tq + D::BYTES;
      const float* rec = reinterpret_cast<const float*>(td + D::BYTES);
      const int* spans = reinterpret_cast<const int*>(rec + 64);
      const bool whole = hl.z <= k0 && hl.w >= k0 + 32 && k0 + 32 <= p.N;
      f32x16_t s = score_block<T, DP>(tq, 0, kf, lane), turn;
      f32x16_t d = score_block<T, DP>(td, 0, vf, lane);
      if constexpr (EXTRA) {
        if (p.cap > 0.f) {
          cap_scores<T, true>(s, turn, p.scale, p.cap);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[r] *= sc2;
            turn[r] = 1.f;
          }
        }
        if (posr) {
          const float slope2 = p.slopes[h] * LOG2E;
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            const int4 ps = *reinterpret_cast<const int4*>(spans + 64 + 8 * q4 + 4 * (lane >> 5));
            s[4 * q4] = fmaf(-slope2, fabsf((float)(ps.x - j)), s[4 * q4]);
            s[4 * q4 + 1] = fmaf(-slope2, fabsf((float)(ps.y - j)), s[4 * q4 + 1]);
            s[4 * q4 + 2] = fmaf(-slope2, fabsf((float)(ps.z - j)), s[4 * q4 + 2]);
            s[4 * q4 + 3] = fmaf(-slope2, fabsf((float)(ps.w - j)), s[4 * q4 + 3]);
          }
        }
      }
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int row = 8 * q4 + 4 * (lane >> 5);
        const float4 lse4 = *reinterpret_cast<const float4*>(rec + row), del4 = *reinterpret_cast<const float4*>(rec + 32 + row);
        const float ls[4] = {lse4.x, lse4.y, lse4.z, lse4.w}, de[4] = {del4.x, del4.y, del4.z, del4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * q4 + e;
          const float pe = __builtin_amdgcn_exp2f(EXTRA ? s[r] - ls[e] : fmaf(s[r], sc2, -ls[e]));
          float ds = pe * (d[r] - de[e]);
          if constexpr (EXTRA) ds *= turn[r];
          s[r] = pe;
          d[r] = ds;
        }
        if (!whole) {
          const int4 lo4 = *reinterpret_cast<const int4*>(spans + row), hi4 = *reinterpret_cast<const int4*>(spans + 32 + row);
          const int lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool on = (unsigned)(j - lo[e]) < (unsigned)(hi[e] - lo[e]);
            s[4 * q4 + e] = on ? s[4 * q4 + e] : 0.f;
            d[4 * q4 + e] = on ? d[4 * q4 + e] : 0.f;
          }
        }
      }
      accum_block<T, DP>(td, 0, s, av, lane);
      accum_block<T, DP>(tq, 0, d, ak, lane);
      if (it + 2 * KW < total) {
        wait_lds();
        issue_nth(it + 2 * KW, buf);
      }
    }
  }
  __syncthreads();
  if (tid < 32) bad[tid] = 0;
  float4 tk[JN], tv[JN];
#pragma unroll
  for (int half = 0; half < 2; ++half) {           // dk, then dv through the same LDS
    join_write<DP>(reinterpret_cast<float*>(mine), half ? av : ak, 1.f, lane);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < JN; ++u) {
      const int idx = tid + u * NT, row = idx / (DP / 4), c4 = idx % (DP / 4);
      const float4 v = join_read<DP, KW>(reinterpret_cast<const float*>(smem), REGION / 4, row, c4);
      if (k0 + row < p.N && !finite4(v)) bad[row] = 1;
      (half ? tv : tk)[u] = v;
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < JN; ++u) {
    const int idx = tid + u * NT, row = idx / (DP / 4), col = idx % (DP / 4) * 4;
    const int64_t r = k0 + row;
    if (r >= p.N || col >= p.dh || bad[row]) continue;
    const float x[4] = {tk[u].x * p.scale, tk[u].y * p.scale, tk[u].z * p.scale, tk[u].w * p.scale};
    const float y[4] = {tv[u].x, tv[u].y, tv[u].z, tv[u].w};
    VecIO<T, 4>::store((T*)p.dk + r * p.ld_dk + kvh * p.dh + col, x);
    VecIO<T, 4>::store((T*)p.dv + r * p.ld_dv + kvh * p.dh + col, y);
  }
  float* xs = reinterpret_cast<float*>(mine);      // (the joined sums have been read)
  for (int row = w; row < 32; row += KW)
    if (bad[row]) span_dkv_key<T>(p, k0 + row, kvh, xs, xs + SPAN_MAX_DH, lane);
}

template <typename T, int DP, int NW>
static int launch_dkv(const SpanParams& p, hipStream_t st) {
  constexpr int RT = NW == 1 || Geo<T, DP>::RB > 128 ? 32 : 64;
  constexpr size_t smem = (size_t)4 * RT * Geo<T, DP>::RB + NW * 2 * SPAN_MAX_DH * sizeof(float);
  const int64_t grid = ((int64_t)p.N + 32 * NW - 1) / (32 * NW) * p.kv_heads;
  NMTGAN_REQUIRE(grid < (1LL << 31), "attn_span_dkv: too many rows");
  // no cap, no slopes: the score is the scaled product itself
  if (p.cap > 0.f || p.slopes || p.scale == 0.f) {
    NMTGAN_TRY(raise_lds(&span_dkv_kernel<T, DP, RT, NW, true>, smem, "attn_span_dkv"));
    hipLaunchKernelGGL((span_dkv_kernel<T, DP, RT, NW, true>), dim3((unsigned)grid), dim3(64 * NW), smem, st, p);
  } else {
    NMTGAN_TRY(raise_lds(&span_dkv_kernel<T, DP, RT, NW, false>, smem, "attn_span_dkv"));
    hipLaunchKernelGGL((span_dkv_kernel<T, DP, RT, NW, false>), dim3((unsigned)grid), dim3(64 * NW), smem, st, p);
  }
  NMTGAN_CHECK_LAUNCH("attn_span_dkv");
  return 0;
}
template <typename T, int DP>
static int launch_dkv_split(const SpanParams& p, hipStream_t st) {
  constexpr int KW = Geo<T, DP>::RB > 256 ? 2 : 4;
  constexpr size_t smem = (size_t)KW * (4 * Dma<T, DP>::BYTES + 2048);
  const int64_t grid = ((int64_t)p.N + 31) / 32 * p.kv_heads;
  if (p.cap > 0.f || p.slopes || p.scale == 0.f) {
    NMTGAN_TRY(raise_lds(&span_dkv_split_kernel<T, DP, KW, true>, smem, "attn_span_dkv"));
    hipLaunchKernelGGL((span_dkv_split_kernel<T, DP, KW, true>), dim3((unsigned)grid), dim3(64 * KW), smem, st, p);
  } else {
    NMTGAN_TRY(raise_lds(&span_dkv_split_kernel<T, DP, KW, false>, smem, "attn_span_dkv"));
    hipLaunchKernelGGL((span_dkv_split_kernel<T, DP, KW, false>), dim3((unsigned)grid), dim3(64 * KW), smem, st, p);
  }
  NMTGAN_CHECK_LAUNCH("attn_span_dkv");
  return 0;
}
template <typename T, int DP>
static int choose_dkv(const SpanParams& p, hipStream_t st) {
  return ((int64_t)p.N + 31) / 32 * p.kv_heads <= SPAN_FEW ? launch_dkv_split<T, DP>(p, st) : launch_dkv<T, DP, 4>(p, st);
}
int span_dkv_tiles(int dtype, const SpanParams& p, hipStream_t st) {
  NMTGAN_DISPATCH_GRAD(dtype, T, {
    if (p.dh <= 32) return choose_dkv<T, 32>(p, st);
    if (p.dh <= 64) return choose_dkv<T, 64>(p, st);
    return choose_dkv<T, 128>(p, st);
  });
  return 0;
}

}  // namespace nmtgan
