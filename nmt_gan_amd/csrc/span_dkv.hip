// Span attention, gradients of keys and values on tiles (span_tiles.h has the formulas and the layout).
#include "span_tiles.h"

namespace nmtgan {

// dk, dv: a workgroup's waves share 32 keys of one key head and take every KW-th of the (row block, head of the group) pairs
// that may see them.  The walk goes by a list of row blocks whose hull meets the keys, made LIST_STEP hulls at a time; an
// entry is 2 block + (every row of the block sees all 32 keys).  Solo: one list for the KW key blocks of a workgroup, each
// wave passing over what does not meet its own.
// Vector arithmetic bounds it where scores are capped and biased (three transcendentals a score): 8192 rows of documents up to
// 3626 long, 8 heads of 64, bf16: 135 us (13 % of the matrix cores' time at the clock it ran at); with the row records read
// where they are used, behind branches of their own, 158 us.  Sentences of at most 50, 2048 rows: 8.8 us.
constexpr int SOLO_BLOCKS = 12;

// hulls of whole chunks of LIST_STEP row blocks, where there are several: a key block passes over the chunks that it does not
// meet (524288 rows of sentences up to 50: both gradients 2.8 ms, 5.4 without)
__global__ __launch_bounds__(256) void span_chunk_kernel(SpanParams p, int nb) {
  __shared__ int lo[4], hi[4];
  int a = 0x7fffffff, b = 0;
#pragma unroll
  for (int u = 0; u < LIST_STEP / 256; ++u) {
    const int at = blockIdx.x * LIST_STEP + 256 * u + threadIdx.x;
    const int4 hl = at < nb ? p.hull[at] : make_int4(0, 0, 0, 0);
    if (hl.y > hl.x) { a = min(a, hl.x); b = max(b, hl.y); }
  }
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    a = min(a, __shfl_xor(a, m));
    b = max(b, __shfl_xor(b, m));
  }
  if ((threadIdx.x & 63) == 0) { lo[threadIdx.x >> 6] = a; hi[threadIdx.x >> 6] = b; }
  __syncthreads();
  if (threadIdx.x == 0)
    p.chunk[blockIdx.x] = make_int2(min(min(lo[0], lo[1]), min(lo[2], lo[3])), max(max(hi[0], hi[1]), max(hi[2], hi[3])));
}
__device__ __forceinline__ bool chunk_meets(const SpanParams& p, int chunk, int a, int b) {
  if (!p.chunk) return true;
  const int2 c = p.chunk[chunk];
  return c.x < b && c.y > a;
}

// appends the blocks of [from, from + LIST_STEP) whose hull meets keys [a, b), in order; returns how many.  All waves call it.
template <int KW>
__device__ __forceinline__ int list_blocks(const SpanParams& p, int from, int nb, int a, int b, int* list, int* count, int w, int lane) {
  constexpr int PER = LIST_STEP / KW / 64;
  const int mine = from + w * (LIST_STEP / KW);
  int4 hl[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int at = mine + 64 * u + lane;
    hl[u] = at < nb ? p.hull[at] : make_int4(0, 0, 0, 0);
  }
  int n = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) n += __popcll(__ballot(hl[u].x < b && hl[u].y > a));
  __syncthreads();                                 // (the last list has been used)
  if (lane == 0) count[w] = n;
  __syncthreads();
  int at = 0, total = 0;
#pragma unroll
  for (int k = 0; k < KW; ++k) {
    if (k < w) at += count[k];
    total += count[k];
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const bool on = hl[u].x < b && hl[u].y > a;
    const unsigned long long mask = __ballot(on);
    if (on)
      list[at + __popcll(mask & ((1ull << lane) - 1))] = 2 * (mine + 64 * u + lane) + (hl[u].z <= a && hl[u].w >= a + 32 && a + 32 <= p.N);
    at += __popcll(mask);
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(total);
}

template <typename T, int DP, int KW, int FORM>
__global__ __launch_bounds__(64 * KW, DP * sizeof(T) <= 128 ? 2 : 1) void span_dkv_split_kernel(SpanParams p) {
  using G = Geo<T, DP>;
  using D = Dma<T, DP>;
  constexpr bool EXTRA = FORM != SPAN_PLAIN, LIBRARY = library_tanh<T, FORM>;
  constexpr int STAGE = 2 * D::BYTES + 1024;      // Q, dO and the records of 32 rows
  constexpr int REGION = 2 * STAGE, NT = 64 * KW, JN = 32 * DP / 4 / NT;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  __shared__ int list[LIST_STEP], count[KW], bad[32];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % p.kv_heads, g = p.heads / p.kv_heads;
  const int nb = (p.M + 31) / 32;
  int k0 = blockIdx.x / p.kv_heads * 32;
  int n_solo = -1, begin = 0;                      // entries of the one list of a solo workgroup, its chunk's first block
  if (p.solo) {
    const int first = k0 / (32 * KW) * (32 * KW);
    int met = 0;
    for (int c = 0; c * LIST_STEP < nb; ++c)
      if (chunk_meets(p, c, first, first + 32 * KW)) {
        begin = c * LIST_STEP;
        ++met;
      }
    if (met <= 1) n_solo = list_blocks<KW>(p, begin, nb, first, first + 32 * KW, list, count, w, lane);
    if (met > 1 || n_solo * g > SOLO_BLOCKS) {
      n_solo = -1;
    } else {
      const int group = first / (32 * KW);        // (not always its first: workgroups go round the shader engines by index)
      if ((k0 - first) / 32 != group % KW) return;
      k0 = first + 32 * w;
    }
  }
  const bool solo = n_solo >= 0;
  const int t0 = solo ? 0 : w, dt = solo ? 1 : KW;
  const int j = k0 + (lane & 31), jc = min(j, p.N - 1);
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
  const bool posr = EXTRA && p.slopes, capped = EXTRA && p.cap > 0.f;
  constexpr int ND = 2 * D::NI + 2 + (EXTRA ? 1 : 0);        // transfers per tile (a record is one)
  auto issue = [&](int b, int h, int buf) {
    const unsigned dst = lds + buf * STAGE;
    dq.issue((const T*)p.q + h * p.dh, p.ldq, b * 32, p.M - b * 32, dst, lane);
    dd.issue((const T*)p.dout + h * p.dh, p.ld_do, b * 32, p.M - b * 32, dst + D::BYTES, lane);
    dma4(lane * 4, p.rec + ((int64_t)h * nb + b) * 64, dst + 2 * D::BYTES);
    dma4(lane * 4, p.spans + (int64_t)b * 64, dst + 2 * D::BYTES + 256);
    if constexpr (EXTRA) dma4(lane * 4, (posr ? p.posr : p.spans) + (int64_t)b * 64, dst + 2 * D::BYTES + 512);
  };

  for (int from = solo ? begin : 0; from < nb; from += LIST_STEP) {
    if (!solo && !chunk_meets(p, from / LIST_STEP, k0, k0 + 32)) continue;
    const int n = solo ? n_solo : list_blocks<KW>(p, from, nb, k0, k0 + 32, list, count, w, lane), total = n * g;
    struct Place { int nth, h; };                  // of a pair: its place in the list, its head
    auto move = [&](Place& at, int by) {
      for (at.nth += by; at.nth >= n; at.nth -= n) ++at.h;
    };
    auto issue_at = [&](const Place& at, int buf) { issue(__builtin_amdgcn_readfirstlane(list[at.nth] >> 1), at.h, buf); };
    Place now{0, kvh * g}, ahead{0, kvh * g};
    if (t0 < total) {
      move(now, t0);
      ahead = now;
      issue_at(now, 0);
    }
    if (t0 + dt < total) {
      move(ahead, dt);
      issue_at(ahead, 1);
    }
    int buf = 0;
    for (int it = t0; it < total; it += dt, buf ^= 1) {
      const int h = now.h, entry = list[now.nth];
      if (it + dt < total) wait_dma<ND>();
      else wait_dma<0>();
      const unsigned char* tq = mine + buf * STAGE;
      const unsigned char* td = tq + D::BYTES;
      const float* rec = reinterpret_cast<const float*>(td + D::BYTES);
      const int* spans = reinterpret_cast<const int*>(rec + 64);
      const bool whole = !solo && (entry & 1);
      float4 lse4[4], del4[4];
      int4 pos4[EXTRA ? 4 : 1];
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int row = 8 * q4 + 4 * (lane >> 5);
        lse4[q4] = *reinterpret_cast<const float4*>(rec + row);
        del4[q4] = *reinterpret_cast<const float4*>(rec + 32 + row);
        if constexpr (EXTRA) pos4[q4] = *reinterpret_cast<const int4*>(spans + 64 + row);
      }
      auto of = [](const auto& v, int e) { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; };
      f32x16_t s = score_block<T, DP>(tq, 0, kf, lane), turn;
      f32x16_t d = score_block<T, DP>(td, 0, vf, lane);
      if (capped) {
        cap_scores<LIBRARY, true>(s, turn, p.scale, p.cap, LIBRARY ? 0.f : p.cap * LOG2E);     // (rec starts there)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] -= of(lse4[r >> 2], r & 3);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = fmaf(s[r], sc2, -of(lse4[r >> 2], r & 3));
      }
      if constexpr (EXTRA) {
        if (posr) {
          const float slope2 = p.slopes[h] * LOG2E;
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(-slope2, fabsf((float)(of(pos4[r >> 2], r & 3) - j)), s[r]);
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(s[r]);
        d[r] = s[r] * (d[r] - of(del4[r >> 2], r & 3));
      }
      if (capped) {
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] *= turned<LIBRARY>(turn[r]);
      }
      if (!whole) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int row = 8 * q4 + 4 * (lane >> 5);
          const int4 lo = *reinterpret_cast<const int4*>(spans + row), hi = *reinterpret_cast<const int4*>(spans + 32 + row);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool on = (unsigned)(j - of(lo, e)) < (unsigned)(of(hi, e) - of(lo, e));
            s[4 * q4 + e] = on ? s[4 * q4 + e] : 0.f;
            d[4 * q4 + e] = on ? d[4 * q4 + e] : 0.f;
          }
        }
      }
      accum_block<T, DP>(td, 0, s, av, lane);
      accum_block<T, DP>(tq, 0, d, ak, lane);
      if (it + dt < total) move(now, dt);
      if (it + 2 * dt < total) {
        move(ahead, dt);
        wait_lds();
        issue_at(ahead, buf);
      }
    }
    if (solo) break;
  }
  if (solo) {
    const unsigned long long off = __ballot(ok && !(all_finite(ak) && all_finite(av)));
    const unsigned again = (unsigned)off | (unsigned)(off >> 32);
    if (ok && !(again >> (lane & 31) & 1)) {
      store_own<T, DP>((T*)p.dk + (int64_t)j * p.ld_dk + kvh * p.dh, ak, result_scale<LIBRARY>(p), p.dh, lane);
      store_own<T, DP>((T*)p.dv + (int64_t)j * p.ld_dv + kvh * p.dh, av, 1.f, p.dh, lane);
    }
    float* xs = reinterpret_cast<float*>(mine);
    for (unsigned left = again; left; left &= left - 1)
      span_dkv_key<T>(p, k0 + __builtin_ctz(left), kvh, xs, xs + SPAN_MAX_DH, lane);
    return;
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
    const float f = result_scale<LIBRARY>(p), x[4] = {tk[u].x * f, tk[u].y * f, tk[u].z * f, tk[u].w * f};
    const float y[4] = {tv[u].x, tv[u].y, tv[u].z, tv[u].w};
    VecIO<T, 4>::store((T*)p.dk + r * p.ld_dk + kvh * p.dh + col, x);
    VecIO<T, 4>::store((T*)p.dv + r * p.ld_dv + kvh * p.dh + col, y);
  }
  float* xs = reinterpret_cast<float*>(mine);      // (the joined sums have been read)
  for (int row = w; row < 32; row += KW)
    if (bad[row]) span_dkv_key<T>(p, k0 + row, kvh, xs, xs + SPAN_MAX_DH, lane);
}

template <typename T, int DP>
static int launch_dkv(SpanParams p, hipStream_t st) {
  constexpr int KW = Geo<T, DP>::RB > 256 ? 2 : 4;
  constexpr size_t smem = (size_t)KW * (4 * Dma<T, DP>::BYTES + 2048);
  const int64_t grid = ((int64_t)p.N + 32 * KW - 1) / (32 * KW) * KW * p.kv_heads;
  NMTGAN_REQUIRE(grid < (1LL << 31), "attn_span_dkv: too many rows");
  p.solo = grid > SPAN_FEW;
  const int nb = (p.M + 31) / 32;
  if (nb > LIST_STEP) {
    hipLaunchKernelGGL(span_chunk_kernel, dim3((nb + LIST_STEP - 1) / LIST_STEP), dim3(256), 0, st, p, nb);
    NMTGAN_CHECK_LAUNCH("attn_span_chunks");
  } else {
    p.chunk = nullptr;
  }
  return with_form<T>(p, [&](auto form) -> int {
    constexpr int FORM = decltype(form)::value;
    NMTGAN_TRY(raise_lds(&span_dkv_split_kernel<T, DP, KW, FORM>, smem, "attn_span_dkv"));
    hipLaunchKernelGGL((span_dkv_split_kernel<T, DP, KW, FORM>), dim3((unsigned)grid), dim3(64 * KW), smem, st, p);
    NMTGAN_CHECK_LAUNCH("attn_span_dkv");
    return 0;
  });
}
int span_dkv_tiles(int dtype, const SpanParams& p, hipStream_t st) {
  NMTGAN_DISPATCH_GRAD(dtype, T, {
    if (p.dh <= 32) return launch_dkv<T, 32>(p, st);
    if (p.dh <= 64) return launch_dkv<T, 64>(p, st);
    return launch_dkv<T, 128>(p, st);
  });
  return 0;
}

}  // namespace nmtgan
