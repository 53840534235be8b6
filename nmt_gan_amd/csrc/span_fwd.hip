// Span attention, forward on tiles (span_tiles.h has the formulas and the layout).
#include "span_tiles.h"

namespace nmtgan {

template <typename T, int DP, int KT, int NW, bool EXTRA>
__global__ __launch_bounds__(64 * NW) void span_fwd_kernel(SpanParams p) {
  using G = Geo<T, DP>;
  constexpr int TB = KT * G::RB, NT = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];          // K[2], V[2], row scratch
  __shared__ int red[NW][2];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int h = blockIdx.x % p.heads, tiles = gridDim.x / p.heads, tile = tiles - 1 - blockIdx.x / p.heads;
  const int kvh = h / (p.heads / p.kv_heads);
  const int i = (tile * NW + w) * 32 + (lane & 31), ic = min(i, p.M - 1);
  const bool ok = i < p.M;
  const int2 sp = ok ? span_of(p, i) : make_int2(0, 0);
  const WaveSpan ws = wave_span(sp);
  const int2 bs = block_span<NW>(ws, red, w);
  const T* K = (const T*)p.k + kvh * p.dh;
  const T* V = (const T*)p.v + kvh * p.dh;
  uint4 own[G::STEPS];
  load_own<T, DP>((const T*)p.q + (int64_t)ic * p.ldq + h * p.dh, ok, p.dh, lane, own);
  const float sc2 = p.scale * LOG2E;
  float slope = 0.f, inv_cap = 0.f;
  int pos = 0;
  if constexpr (EXTRA) {
    if (p.slopes) { slope = p.slopes[h]; pos = pos_of(p, ic); }
    if (p.cap > 0.f) inv_cap = 1.f / p.cap;
  }
  f32x16_t acc[G::DB];
  clear(acc);
  float m = -INFINITY, l = 0.f;
  const unsigned len = (unsigned)(sp.y - sp.x);

  Stage<T, DP, KT, NT> sk, sv;
  const int nt = bs.y > bs.x ? (bs.y - bs.x + KT - 1) / KT : 0;
  if (nt > 0) {
    sk.load(K, p.ldk, bs.x, bs.y, p.dh, tid);
    sv.load(V, p.ldv, bs.x, bs.y, p.dh, tid);
    sk.store(smem, tid);
    sv.store(smem + 2 * TB, tid);
  }
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    const int j0 = bs.x + t * KT;
    if (t + 1 < nt) {
      sk.load(K, p.ldk, j0 + KT, bs.y, p.dh, tid);
      sv.load(V, p.ldv, j0 + KT, bs.y, p.dh, tid);
    }
    if (j0 < ws.hi && j0 + KT > ws.lo) {
      const unsigned char* tk = smem + (t & 1) * TB;
      const unsigned char* tv = smem + (2 + (t & 1)) * TB;
      f32x16_t s[KT / 32];
#pragma unroll
      for (int kb = 0; kb < KT / 32; ++kb) s[kb] = score_block<T, DP>(tk, kb, own, lane);
      if constexpr (EXTRA) {
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float turn;
            s[kb][r] = score2<T>(p, s[kb][r], inv_cap, slope, pos, j0 + 32 * kb + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), turn);
          }
      }
      const bool flip = !EXTRA && sc2 < 0.f;      // the largest score is the smallest product
      if (!(j0 >= ws.all_lo && j0 + KT <= ws.all_hi)) {
        const float out = flip ? INFINITY : -INFINITY;
        const int base = j0 + 4 * (lane >> 5) - sp.x;
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            s[kb][r] = (unsigned)(base + 32 * kb + 8 * (r >> 2) + (r & 3)) < len ? s[kb][r] : out;
      }
      float mx;
      if (flip) {
        mx = INFINITY;
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fminf(mx, s[kb][r]);
      } else {
        mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
      }
      const float f = EXTRA ? 1.f : sc2;
      mx = both_halves_max(EXTRA ? mx : (isinf(mx) ? -INFINITY : mx * f));
      const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn;
      if (__any(mn > m)) {
        const float c = __builtin_amdgcn_exp2f(m - mu);
        l *= c;
#pragma unroll
        for (int db = 0; db < G::DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= c;
        m = mn;
      }
#pragma unroll
      for (int kb = 0; kb < KT / 32; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[kb][r] = __builtin_amdgcn_exp2f(EXTRA ? s[kb][r] - mu : fmaf(s[kb][r], f, -mu));
          l += s[kb][r];
        }
        accum_block<T, DP>(tv, kb, s[kb], acc, lane);
      }
    }
    if (t + 1 < nt) {
      sk.store(smem + ((t + 1) & 1) * TB, tid);
      sv.store(smem + (2 + ((t + 1) & 1)) * TB, tid);
    }
    __syncthreads();
  }
  l = both_halves_sum(l);
  const bool some = sp.y > sp.x;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  // a product of a zero probability with an infinity or NaN of a row this row does not see: such rows are done again one
  // by one (as are rows that are not finite by right)
  const unsigned long long bad = __ballot(some && !(all_finite(acc) && l < INFINITY));
  if (ok && !((bad >> (lane & 31) | bad >> ((lane & 31) + 32)) & 1)) {
    T* o = (T*)p.out + (int64_t)i * p.ldo + h * p.dh;
    if (!some || l == 0.f) clear(acc);
    store_own<T, DP>(o, acc, inv, p.dh, lane);
    if (p.lse && lane < 32) p.lse[(int64_t)i * p.heads + h] = !some || l == 0.f ? -INFINITY : m * LN2 + logf(l);
  }
  if (bad) {
    float* x = reinterpret_cast<float*>(smem + 4 * TB) + w * SPAN_MAX_DH;
    for (unsigned left = (unsigned)bad | (unsigned)(bad >> 32); left; left &= left - 1)
      span_fwd_row<T>(p, (tile * NW + w) * 32 + __builtin_ctz(left), h, x, lane);
  }
}


template <typename T, int DP, int NW>
static int launch_fwd(const SpanParams& p, hipStream_t st) {
  constexpr int RT = NW == 1 || Geo<T, DP>::RB > 128 ? 32 : 64;
  constexpr size_t smem = (size_t)4 * RT * Geo<T, DP>::RB + NW * 1 * SPAN_MAX_DH * sizeof(float);
  const int64_t grid = ((int64_t)p.M + 32 * NW - 1) / (32 * NW) * p.heads;
  NMTGAN_REQUIRE(grid < (1LL << 31), "attn_span: too many rows");
  // no cap, no slopes: the score is the scaled product itself
  if (p.cap > 0.f || p.slopes || p.scale == 0.f) {
    NMTGAN_TRY(raise_lds(&span_fwd_kernel<T, DP, RT, NW, true>, smem, "attn_span"));
    hipLaunchKernelGGL((span_fwd_kernel<T, DP, RT, NW, true>), dim3((unsigned)grid), dim3(64 * NW), smem, st, p);
  } else {
    NMTGAN_TRY(raise_lds(&span_fwd_kernel<T, DP, RT, NW, false>, smem, "attn_span"));
    hipLaunchKernelGGL((span_fwd_kernel<T, DP, RT, NW, false>), dim3((unsigned)grid), dim3(64 * NW), smem, st, p);
  }
  NMTGAN_CHECK_LAUNCH("attn_span");
  return 0;
}
template <typename T, int DP>
static int choose_fwd(const SpanParams& p, hipStream_t st) {
  return ((int64_t)p.M + 31) / 32 * p.heads <= SPAN_FEW_WAVES ? launch_fwd<T, DP, 1>(p, st) : launch_fwd<T, DP, 4>(p, st);
}
int span_fwd_tiles(int dtype, const SpanParams& p, hipStream_t st) {
  NMTGAN_DISPATCH_OP(dtype, T, {
    if (p.dh <= 32) return choose_fwd<T, 32>(p, st);
    if (p.dh <= 64) return choose_fwd<T, 64>(p, st);
    return choose_fwd<T, 128>(p, st);
  });
  return 0;
}

}  // namespace nmtgan
