// Span attention, gradient of the queries on tiles (span_tiles.h has the formulas and the layout).
#include "span_tiles.h"

namespace nmtgan {

// dq.  delta = dout . out carries the rounding of a 16-bit `out`, which shows where a row has few keys that count; the sum
// of p dp over the walk does not.  So the walk runs with the former and corrects at the end: with c = p (1 - t^2),
//   dq / scale = sum c (dp - delta) k = sum c (dp - delta16) k + (delta16 - delta) sum c k,
// the second sum riding on the same turned K fragments.  The dk/dv kernel gets the corrected delta.  (8192 rows of documents up to
// 3626 long, 8 heads of 64, capped and biased, bf16: 127 us, 111 without the correction and with 1.5 times the error that
// rounding the results alone leaves in dq and dk; taking every span twice instead: 190 us.)
template <typename T, int DP, int KW, int FORM>
__global__ __launch_bounds__(64 * KW, DP * sizeof(T) <= 128 ? 2 : 1) void span_dq_split_kernel(SpanParams p) {
  using G = Geo<T, DP>;
  using D = Dma<T, DP>;
  constexpr bool EXTRA = FORM != SPAN_PLAIN, LIBRARY = library_tanh<T, FORM>;
  constexpr int REGION = 3 * D::BYTES, NT = 64 * KW, JN = 32 * DP / 4 / NT;      // two K tiles and one V tile per wave
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ float s_sum[KW][32], xs[KW][2][SPAN_MAX_DH];
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
  auto issue_k = [&](int t, int buf) { dk.issue(K, p.ldk, ws.lo + 32 * t, ws.hi - ws.lo - 32 * t, lds + buf * D::BYTES, lane); };
  auto issue_v = [&](int t) { dv.issue(V, p.ldv, ws.lo + 32 * t, ws.hi - ws.lo - 32 * t, lds + 2 * D::BYTES, lane); };
  uint4 own[G::STEPS], dout[G::STEPS];
  load_own<T, DP>((const T*)p.q + (int64_t)ic * p.ldq + h * p.dh, ok, p.dh, lane, own);
  load_own<T, DP>((const T*)p.dout + (int64_t)ic * p.ld_do + h * p.dh, ok, p.dh, lane, dout);
  const float ls = ok ? p.lse[(int64_t)i * p.heads + h] : 0.f;
  const float lse2 = ls == -INFINITY ? 0.f : ls * LOG2E, sc2 = p.scale * LOG2E;
  float delta = 0.f;
  {
    uint4 o[G::STEPS];
    load_own<T, DP>((const T*)p.out + (int64_t)ic * p.ldo + h * p.dh, ok, p.dh, lane, o);
#pragma unroll
    for (int s = 0; s < G::STEPS; ++s) delta += chunk_dot<T>(o[s], dout[s]);
    delta = sp.y > sp.x ? both_halves_sum(delta) : 0.f;
  }
  float slope2 = 0.f;
  int pos = 0;
  if constexpr (EXTRA) {
    if (p.slopes) { slope2 = p.slopes[h] * LOG2E; pos = pos_of(p, ic); }
  }
  constexpr bool FIX = sizeof(T) == 2;
  f32x16_t acc[G::DB], ck[FIX ? G::DB : 1];
  clear(acc);
  clear(ck);
  const unsigned len = (unsigned)(sp.y - sp.x);
  const bool capped = EXTRA && p.cap > 0.f;
  float sum = 0.f;
  if (t0 < nt) {
    issue_k(t0, 0);
    issue_v(t0);
  }
  if (t0 + dt < nt) issue_k(t0 + dt, 1);
  int buf = 0;
  for (int t = t0; t < nt; t += dt, buf ^= 1) {
    const int j0 = ws.lo + 32 * t;
    if (t + dt < nt) wait_dma<D::NI>();           // the next K may still be under way
    else wait_dma<0>();
    const unsigned char* tk = mine + buf * D::BYTES;
    f32x16_t s = score_block<T, DP>(tk, 0, own, lane), turn = s;
    f32x16_t d = score_block<T, DP>(mine + 2 * D::BYTES, 0, dout, lane);
    if (t + dt < nt) {
      wait_lds();
      issue_v(t + dt);
    }
    if (__any(sp.x < j0 + 32 && sp.y > j0)) {
      if (capped) {
        cap_scores<LIBRARY, true>(s, turn, p.scale, p.cap, lse2);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], sc2, -lse2);
      }
      const int first = j0 + 4 * (lane >> 5);
      if (EXTRA && p.slopes) {
        const float away = (float)(pos - first);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(-slope2, fabsf(away - (float)(8 * (r >> 2) + (r & 3))), s[r]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]);
      if (!(j0 >= ws.all_lo && j0 + 32 <= ws.all_hi)) {      // what lies outside the rows' spans counts as zero
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const bool on = (unsigned)(first - sp.x + 8 * (r >> 2) + (r & 3)) < len;
          s[r] = on ? s[r] : 0.f;
          d[r] = on ? d[r] : 0.f;
        }
      }
      if constexpr (FIX) {
#pragma unroll
        for (int r = 0; r < 16; ++r) sum = fmaf(s[r], d[r], sum);
      }
      if (capped) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= turned<LIBRARY>(turn[r]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) d[r] = s[r] * (d[r] - delta);
      if constexpr (FIX) accum_two<T, DP>(tk, d, s, acc, ck, lane);
      else accum_block<T, DP>(tk, 0, d, acc, lane);
    }
    if (t + 2 * dt < nt) {
      wait_lds();
      issue_k(t + 2 * dt, buf);
    }
  }
  if constexpr (FIX) {
    const float given = delta;
    sum = both_halves_sum(sum);
    delta = sum;
    if (!solo) {
      if (lane < 32) s_sum[w][lane] = sum;
      __syncthreads();
      delta = s_sum[0][lane & 31];
#pragma unroll
      for (int k = 1; k < KW; ++k) delta += s_sum[k][lane & 31];
    }
    if (!(sp.y > sp.x)) delta = 0.f;
    const float off = given - delta;
#pragma unroll
    for (int db = 0; db < G::DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] = fmaf(off, ck[db][r], acc[db][r]);
  }
  // what the dk/dv kernel reads of these rows: a record per head, and once for all heads the spans and their hull
  if (lane < 32 && (solo || w == 0) && tile * 32 < p.M) {
    float* const at = delta_at(p, i, h);
    at[-32] = capped && !LIBRARY ? lse2 - p.cap * LOG2E : lse2;      // (where the capped score starts)
    at[0] = delta;
    if (h == 0) {
      p.spans[(int64_t)tile * 64 + lane] = sp.x;
      p.spans[(int64_t)tile * 64 + 32 + lane] = sp.y;
      if (p.slopes) p.posr[(int64_t)tile * 64 + lane] = ok ? pos_of(p, i) : 0;
      if (lane == 0) p.hull[tile] = make_int4(ws.lo, ws.hi, ws.all_lo, ws.all_hi);
    }
  }
  if (solo) {
    const bool some = sp.y > sp.x;
    const unsigned long long off = __ballot(some && !all_finite(acc));
    const unsigned again = (unsigned)off | (unsigned)(off >> 32);
    if (ok && !(again >> (lane & 31) & 1)) {
      if (!some) clear(acc);
      store_own<T, DP>((T*)p.dq + (int64_t)i * p.ld_dq + h * p.dh, acc, result_scale<LIBRARY>(p), p.dh, lane);
    }
    __threadfence_block();
    for (unsigned left = again; left; left &= left - 1)
      span_dq_row<T>(p, tile * 32 + __builtin_ctz(left), h, xs[w][0], xs[w][1], lane);
    return;
  }
  if (tid < 32) {
    bad[tid] = 0;
    seen[tid] = sp.y > sp.x;
  }
  join_write<DP>(reinterpret_cast<float*>(mine), acc, 1.f, lane);
  __syncthreads();
  float4 tot[JN];
#pragma unroll
  for (int u = 0; u < JN; ++u) {
    const int idx = tid + u * NT, row = idx / (DP / 4), c4 = idx % (DP / 4), r = tile * 32 + row;
    tot[u] = join_read<DP, KW>(reinterpret_cast<const float*>(smem), REGION / 4, row, c4);
    if (r >= p.M) continue;
    if (!seen[row]) tot[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    else if (!finite4(tot[u])) bad[row] = 1;
  }
  __threadfence_block();                          // delta is read again by rows that are done one by one
  __syncthreads();
#pragma unroll
  for (int u = 0; u < JN; ++u) {
    const int idx = tid + u * NT, row = idx / (DP / 4), col = idx % (DP / 4) * 4, r = tile * 32 + row;
    if (r >= p.M || col >= p.dh || bad[row]) continue;
    const float f = result_scale<LIBRARY>(p), x[4] = {tot[u].x * f, tot[u].y * f, tot[u].z * f, tot[u].w * f};
    VecIO<T, 4>::store((T*)p.dq + (int64_t)r * p.ld_dq + h * p.dh + col, x);
  }
  for (int row = w; row < 32; row += KW)
    if (bad[row]) span_dq_row<T>(p, tile * 32 + row, h, xs[w][0], xs[w][1], lane);
}

template <typename T, int DP>
static int launch_dq(SpanParams p, hipStream_t st) {
  constexpr int KW = Geo<T, DP>::RB > 256 ? 2 : 4;
  constexpr size_t smem = (size_t)KW * 3 * Dma<T, DP>::BYTES;
  const int64_t grid = ((int64_t)p.M + 32 * KW - 1) / (32 * KW) * KW * p.heads;
  NMTGAN_REQUIRE(grid < (1LL << 31), "attn_span_dq: too many rows");
  p.solo = grid > SPAN_FEW;
  return with_form<T>(p, [&](auto form) -> int {
    constexpr int FORM = decltype(form)::value;
    NMTGAN_TRY(raise_lds(&span_dq_split_kernel<T, DP, KW, FORM>, smem, "attn_span_dq"));
    hipLaunchKernelGGL((span_dq_split_kernel<T, DP, KW, FORM>), dim3((unsigned)grid), dim3(64 * KW), smem, st, p);
    NMTGAN_CHECK_LAUNCH("attn_span_dq");
    return 0;
  });
}
int span_dq_tiles(int dtype, const SpanParams& p, hipStream_t st) {
  NMTGAN_DISPATCH_GRAD(dtype, T, {
    if (p.dh <= 32) return launch_dq<T, 32>(p, st);
    if (p.dh <= 64) return launch_dq<T, 64>(p, st);
    return launch_dq<T, 128>(p, st);
  });
  return 0;
}

}  // namespace nmtgan
