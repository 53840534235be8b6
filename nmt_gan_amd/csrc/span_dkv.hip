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
        const float ls = p.lse[(int64_t)i * p.heads + h];
        r_lse = ls == -INFINITY ? 0.f : ls * LOG2E;
        r_delta = p.delta[(int64_t)i * p.heads + h];
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
static int choose_dkv(const SpanParams& p, hipStream_t st) {
  return ((int64_t)p.N + 31) / 32 * p.kv_heads <= SPAN_FEW_WAVES ? launch_dkv<T, DP, 1>(p, st) : launch_dkv<T, DP, 4>(p, st);
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
