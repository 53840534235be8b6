// Span attention, forward on tiles (span_tiles.h has the formulas and the layout).
#include "span_tiles.h"

namespace nmtgan {

// One pass over the keys with the running maximum and sum of the softmax.  Bound by vector arithmetic (an exponential, with a
// cap a second one and a reciprocal, per score) and, where one long document holds most of the work, by its last rows:
//   8192 rows of documents up to 3626 long, 8 heads of 64, capped and biased, bf16: 99 us (60 % of the vector units' time)
//   5000 rows of prompts up to 2390 long, 8 heads of 128 over 2 key heads, fp16: 47 us, 1.4 waves a SIMD on average of the 2
//     that fit; eight waves a workgroup instead of four: 63 us (and 90 and 8.8 us for the two other cases)
//   2048 rows of sentences up to 50 long, 8 heads of 64, bf16: 7.5 us, most of it launch and first loads
template <typename T, int DP, int KW, int FORM>
__global__ __launch_bounds__(64 * KW, DP * sizeof(T) <= 256 ? 2 : 1) void span_fwd_split_kernel(SpanParams p) {
  using G = Geo<T, DP>;
  using D = Dma<T, DP>;
  constexpr bool EXTRA = FORM != SPAN_PLAIN, LIBRARY = library_tanh<T, FORM>;
  // one K and one V tile per wave: the next K is under way during the softmax and the second product, the next V during
  // the first product and the softmax, and the small footprint buys waves to hide the rest behind
  constexpr int REGION = 2 * D::BYTES > 32 * DP * 4 ? 2 * D::BYTES : 32 * DP * 4, NT = 64 * KW, JN = 32 * DP / 4 / NT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ float s_m[KW][32], s_l[KW][32], xs[KW][SPAN_MAX_DH];
  __shared__ int bad[32], seen[32], s_hull[KW];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = blockIdx.x % p.heads, last = gridDim.x / p.heads - 1;
  const int kvh = h / (p.heads / p.kv_heads);
  int tile = last - (int)(blockIdx.x / p.heads);
  const bool solo = p.solo && group_is_short<KW>(p, tile / KW * KW, s_hull, w, lane);
  if (solo) {
    const int group = tile / KW;                  // (not always its first: workgroups go round the shader engines by index)
    if (tile % KW != group % KW) return;
    tile = group * KW + w;
  }
  const int i = tile * 32 + (lane & 31), ic = min(i, p.M - 1);
  const bool ok = i < p.M;
  const int2 sp = ok ? span_of(p, i) : make_int2(0, 0);
  const WaveSpan ws = wave_span(sp);
  const int t0 = solo ? 0 : w, dt = solo ? 1 : KW;
  const T* K = (const T*)p.k + kvh * p.dh;
  const T* V = (const T*)p.v + kvh * p.dh;
  unsigned char* mine = smem + w * REGION;
  const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) void*)mine);
  D dk, dv;
  dk.init(p.ldk, p.dh, lane);
  dv.init(p.ldv, p.dh, lane);
  const int nt = ws.hi > ws.lo ? (ws.hi - ws.lo + 31) / 32 : 0;
  auto issue_k = [&](int t) { dk.issue(K, p.ldk, ws.lo + 32 * t, ws.hi - ws.lo - 32 * t, lds, lane); };
  auto issue_v = [&](int t) { dv.issue(V, p.ldv, ws.lo + 32 * t, ws.hi - ws.lo - 32 * t, lds + D::BYTES, lane); };
  uint4 own[G::STEPS];
  load_own<T, DP>((const T*)p.q + (int64_t)ic * p.ldq + h * p.dh, ok, p.dh, lane, own);
  if (t0 < nt) {
    issue_k(t0);
    issue_v(t0);
  }
  const float sc2 = p.scale * LOG2E;
  float slope2 = 0.f;
  int pos = 0;
  if constexpr (EXTRA) {
    if (p.slopes) { slope2 = p.slopes[h] * LOG2E; pos = pos_of(p, ic); }
  }
  f32x16_t acc[G::DB];
  clear(acc);
  float m = -INFINITY, l = 0.f;
  const unsigned len = (unsigned)(sp.y - sp.x);
  const bool few = len <= SPAN_SHORT && len > 0, any_few = !LIBRARY && __any(few);

  for (int t = t0; t < nt; t += dt) {
    const int j0 = ws.lo + 32 * t;
    const bool more = t + dt < nt;
    wait_dma<D::NI>();                            // V may still be under way
    f32x16_t s = score_block<T, DP>(mine, 0, own, lane);
    if (more) {
      wait_lds();
      issue_k(t + dt);
    }
    const bool met = __any(sp.x < j0 + 32 && sp.y > j0);
    if (met) {
      const int first = j0 + 4 * (lane >> 5);
      if constexpr (EXTRA) {
        if (p.cap > 0.f) {
          if (any_few) cap_scores_fine(s, p.scale, p.cap, few);
          else cap_scores<LIBRARY, false>(s, s, p.scale, p.cap, 0.f);
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] *= sc2;
        }
        if (p.slopes) {
          const float away = (float)(pos - first);
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(-slope2, fabsf(away - (float)(8 * (r >> 2) + (r & 3))), s[r]);
        }
      }
      const bool flip = !EXTRA && sc2 < 0.f;      // the largest score is the smallest product
      if (!(j0 >= ws.all_lo && j0 + 32 <= ws.all_hi)) {
        const float out = flip ? INFINITY : -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = (unsigned)(first - sp.x + 8 * (r >> 2) + (r & 3)) < len ? s[r] : out;
      }
      float mx = flip ? INFINITY : -INFINITY;
      if (flip) {
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fminf(mx, s[r]);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
      }
      mx = both_halves_max(EXTRA ? mx : (isinf(mx) ? -INFINITY : mx * sc2));
      // the reference point follows the maximum only when it falls 2^8 behind: probabilities up to 256 fit every type
      if (__any(mx > m + 8.f)) {
        const float mn = fmaxf(m, mx), c = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        l *= c;
#pragma unroll
        for (int db = 0; db < G::DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= c;
        m = mn;
      }
      const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(EXTRA ? s[r] - mu : fmaf(s[r], sc2, -mu));
        l += s[r];
      }
    }
    if (more) wait_dma<D::NI>();                  // the next K may still be under way
    else wait_dma<0>();
    if (met) accum_block<T, DP>(mine + D::BYTES, 0, s, acc, lane);
    if (more) {
      wait_lds();
      issue_v(t + dt);
    }
  }
  l = both_halves_sum(l);
  const bool some = sp.y > sp.x;
  if (solo) {
    const unsigned long long off = __ballot(some && !(all_finite(acc) && l < INFINITY));
    const unsigned again = (unsigned)off | (unsigned)(off >> 32);
    if (ok && !(again >> (lane & 31) & 1)) {
      if (!some) clear(acc);
      store_own<T, DP>((T*)p.out + (int64_t)i * p.ldo + h * p.dh, acc, l == 0.f ? 0.f : 1.f / l, p.dh, lane);
      if (p.lse && lane < 32) p.lse[(int64_t)i * p.heads + h] = !some || l == 0.f ? -INFINITY : m * LN2 + logf(l);
    }
    for (unsigned left = again; left; left &= left - 1) span_fwd_row<T>(p, tile * 32 + __builtin_ctz(left), h, xs[w], lane);
    return;
  }
  if (lane < 32) { s_m[w][lane] = m; s_l[w][lane] = l; }
  if (tid < 32) {
    bad[tid] = 0;
    seen[tid] = sp.y > sp.x;
  }
  __syncthreads();
  float mt = s_m[0][lane & 31];
#pragma unroll
  for (int k = 1; k < KW; ++k) mt = fmaxf(mt, s_m[k][lane & 31]);
  const float mu = mt == -INFINITY ? 0.f : mt;
  join_write<DP>(reinterpret_cast<float*>(mine), acc, __builtin_amdgcn_exp2f(m - mu), lane);
  __syncthreads();
  float4 sum[JN];
  float inv[JN];
#pragma unroll
  for (int u = 0; u < JN; ++u) {
    const int idx = tid + u * NT, row = idx / (DP / 4), c4 = idx % (DP / 4), r = tile * 32 + row;
    float mr = s_m[0][row], lr = 0.f;
#pragma unroll
    for (int k = 1; k < KW; ++k) mr = fmaxf(mr, s_m[k][row]);
    const float mur = mr == -INFINITY ? 0.f : mr;
#pragma unroll
    for (int k = 0; k < KW; ++k) lr += s_l[k][row] * __builtin_amdgcn_exp2f(s_m[k][row] - mur);
    sum[u] = join_read<DP, KW>(reinterpret_cast<const float*>(smem), REGION / 4, row, c4);
    inv[u] = 0.f;
    if (r >= p.M) continue;
    if (seen[row]) {
      inv[u] = lr == 0.f ? 0.f : 1.f / lr;
      if (!(finite4(sum[u]) && lr < INFINITY)) bad[row] = 1;
    } else {
      sum[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      lr = 0.f;
    }
    if (p.lse && c4 == 0) p.lse[(int64_t)r * p.heads + h] = lr == 0.f ? -INFINITY : mur * LN2 + logf(lr);
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < JN; ++u) {
    const int idx = tid + u * NT, row = idx / (DP / 4), col = idx % (DP / 4) * 4, r = tile * 32 + row;
    if (r >= p.M || col >= p.dh || bad[row]) continue;
    const float x[4] = {sum[u].x * inv[u], sum[u].y * inv[u], sum[u].z * inv[u], sum[u].w * inv[u]};
    VecIO<T, 4>::store((T*)p.out + (int64_t)r * p.ldo + h * p.dh + col, x);
  }
  // a product of a zero probability with an infinity or NaN of a row this row does not see: such rows are done again one
  // by one (as are rows that are not finite by right)
  for (int row = w; row < 32; row += KW)
    if (bad[row]) span_fwd_row<T>(p, tile * 32 + row, h, xs[w], lane);
}

template <typename T, int DP>
static int launch_fwd(SpanParams p, hipStream_t st) {
  constexpr int KW = Geo<T, DP>::RB > 256 ? 2 : 4;
  constexpr size_t smem = (size_t)KW * std::max(2 * Dma<T, DP>::BYTES, 32 * DP * 4);
  const int64_t grid = ((int64_t)p.M + 32 * KW - 1) / (32 * KW) * KW * p.heads;
  NMTGAN_REQUIRE(grid < (1LL << 31), "attn_span: too many rows");
  p.solo = grid > SPAN_FEW;
  return with_form<T>(p, [&](auto form) -> int {
    constexpr int FORM = decltype(form)::value;
    NMTGAN_TRY(raise_lds(&span_fwd_split_kernel<T, DP, KW, FORM>, smem, "attn_span"));
    hipLaunchKernelGGL((span_fwd_split_kernel<T, DP, KW, FORM>), dim3((unsigned)grid), dim3(64 * KW), smem, st, p);
    NMTGAN_CHECK_LAUNCH("attn_span");
    return 0;
  });
}
int span_fwd_tiles(int dtype, const SpanParams& p, hipStream_t st) {
  NMTGAN_DISPATCH_OP(dtype, T, {
    if (p.dh <= 32) return launch_fwd<T, 32>(p, st);
    if (p.dh <= 64) return launch_fwd<T, 64>(p, st);
    return launch_fwd<T, 128>(p, st);
  });
  return 0;
}

}  // namespace nmtgan
