// Softmax cross entropy of hidden rows against a vocabulary table (formulas: xent.hip), the direct form: few launches and
// 32 x 32 wave tiles, operands read from the caches in the layout they have and multiplied in fp32 (v_mfma_f32_32x32x2,
// no rounding of d(logits); logits of 16-bit operands on their own matrix instructions).  For little work, which on 256 x 256 tiles is launches, layout
// changes and tiles that fill a few of the 256 CUs, and for fp32 gradients:
//   forward: z^T by tiles with (max, sum exp) per row and 32 entries, then the finish kernel
//   gradient: z again and y = dz / g [M][V] in fp32, then dh and dw side by side in one launch
// Bound by the rate at which the caches answer: 8 to 11 flop per byte loaded, 44 TFLOP/s of the fp32 matrix cores' 154 in the
// products of 3200 rows over 32000 entries, d = 512; of few rows by w and dw in memory: 8 rows over 32000 entries, d = 512,
// bf16, 11 us for the logits (3 TB/s) and 36 us for both products (1.8 TB/s); of little work by the launches: 13 us for the
// gradient's two at 97 x 509 x 64, called back to back.
// Which k goes into which slot of a product is free as long as both operands agree: lane half hl takes k = 8 s + 4 hl + t
// in product t of step s, so that an operand with its k dimension in memory order is read by 16 bytes.
#include "common.h"
#include "kernels.h"

namespace nmtgan {

// products of two operands' 16-byte chunks, one per lane half
template <typename T>
__device__ __forceinline__ f32x16_t mul_chunk(const uint4& a, const uint4& b, f32x16_t c) {
  if constexpr (sizeof(T) == 2) {
    return mfma16<T>(a, b, c);
  } else {
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}
__device__ __forceinline__ f32x16_t zero16() {
  f32x16_t c;
#pragma unroll
  for (int r = 0; r < 16; ++r) c[r] = 0.f;
  return c;
}
__device__ __forceinline__ float halves_sum(float v) { return v + __shfl_xor(v, 32); }

// z^T: C rows = 32 entries, C columns = 32 hidden rows, so that a lane has 16 logits of one row.  A workgroup takes four
// entry tiles of a row tile, a wave each.  GRAD: y = dz / g into y[M][Vp] (zero behind V and in rows
// without a gradient), the rows' g into coef.
template <typename T, bool GRAD>
__global__ __launch_bounds__(256) void xent_direct_z_kernel(XentDirect p) {
  const int across = (p.Vp + 127) / 128;
  const int lane = threadIdx.x & 63, hl = lane >> 5, tile = blockIdx.x % across * 4 + (threadIdx.x >> 6), e0 = tile * 32;
  const int row = blockIdx.x / across * 32 + (lane & 31), rc = min(row, p.M - 1);
  const int label = p.labels[rc];
  const bool used = label >= 0 && label < p.V_all;
  float coef = 0.f;
  if constexpr (GRAD) {
    coef = used ? (p.grad_row ? p.grad_row[rc] : 1.f) : 0.f;
    if (tile == 0 && hl == 0 && row < p.M) p.coef[row] = coef;
  }
  if (e0 >= p.Vp) return;
  const T* a = (const T*)p.w + (int64_t)min(e0 + (lane & 31), p.V - 1) * p.ldw;
  const T* b = (const T*)p.h + (int64_t)rc * p.ldh;
  f32x16_t z = zero16();
  constexpr int U = 8, E = 16 / (int)sizeof(T);    // a batch of 16 E k, the next one under way while it is multiplied
  uint4 x[U], y[U];
  auto fetch = [&](int k) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(k + E * (2 * u + hl), p.d - E);
      x[u] = *reinterpret_cast<const uint4*>(a + at);
      y[u] = *reinterpret_cast<const uint4*>(b + at);
    }
  };
  fetch(0);
  for (int k = 0; k < p.d; k += 2 * E * U) {
    uint4 f[U], g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool ok = k + E * (2 * u + hl) < p.d;
      f[u] = ok ? x[u] : make_uint4(0, 0, 0, 0);
      g[u] = ok ? y[u] : make_uint4(0, 0, 0, 0);
    }
    if (k + 2 * E * U < p.d) fetch(k + 2 * E * U);
#pragma unroll
    for (int u = 0; u < U; ++u) z = mul_chunk<T>(f[u], g[u], z);
  }
  if constexpr (GRAD) {
    if (row >= p.M) return;
    const float lse2 = p.lse[row] * 1.44269504088896341f;
    float* out = p.y + (int64_t)row * p.Vp + e0 + 4 * hl;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int e = e0 + 8 * g + 4 * hl;
      if (e >= p.Vp) continue;
      float o[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float q = p.first + e + t == label ? p.high + p.low : p.low;
        o[t] = __builtin_amdgcn_exp2f(fmaf(z[4 * g + t], 1.44269504088896341f, -lse2)) - q;
        if (coef == 0.f || e + t >= p.V) o[t] = 0.f;
      }
      VecIO<float, 4>::store(out + 8 * g, o);
    }
  } else {
    const int left = p.V - e0 - 4 * hl;            // entries of the lane: 8 (r / 4) + r % 4 < left
    float mx = -INFINITY, zs = 0.f, s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool on = 8 * (r >> 2) + (r & 3) < left;
      zs += on ? z[r] : 0.f;
      z[r] = on ? z[r] : -INFINITY;
      mx = fmaxf(mx, z[r]);
    }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mu2 = mx == -INFINITY ? 0.f : mx * 1.44269504088896341f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += __builtin_amdgcn_exp2f(fmaf(z[r], 1.44269504088896341f, -mu2));
    s = halves_sum(s);
    zs = halves_sum(zs);
    if (hl == 0 && row < p.M) {
      p.stats[(int64_t)tile * p.M + row] = make_float2(mx, s);
      if (p.zsum) p.zsum[(int64_t)tile * p.M + row] = zs;
    }
  }
}

// dh = g (y w) by the first n_dh workgroups, one slice of the entries of a tile of 32 rows x 32 NC columns each, which 16 waves
// divide; dw = y^T (g h) by the others, one slice of the rows of 1, 4 or 16 tiles of 32 entries x 32 NC columns, which 16, 4 or 1
// waves divide.  A lane has NC neighbouring columns: 2 make rows come and go in whole cache lines and use a value of y twice (1
// row over 31989 entries, d = 768, bf16: 46 us against 61), 1 fills more CUs where tiles are few (97 x 509 x 64, fp32: 7 us
// against 10).  Waves are joined in order through LDS, one element per thread; of several slices each leaves
// its part.  Loads go to clamped addresses and are selected afterwards: under a condition each, they would not be in flight
// together.
template <typename T, int NC>
__global__ __launch_bounds__(1024) void xent_direct_grads_kernel(XentDirect p) {
  __shared__ float part[16][1024];
  const int lane = threadIdx.x & 63, hl = lane >> 5, w = threadIdx.x >> 6;
  f32x16_t c[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) c[k] = zero16();
  constexpr int WIDE = 32 * NC;
  const int across = (p.d + WIDE - 1) / WIDE;
  const int reg = threadIdx.x >> 6, sub = 8 * (reg >> 2) + 4 * hl + (reg & 3);      // the element joined by this thread
  auto put = [&](int half) {
#pragma unroll
    for (int r = 0; r < 16; ++r) part[w][r * 64 + lane] = c[half][r];
    __syncthreads();
  };
  if ((int)blockIdx.x < p.n_dh) {
    const int slice = blockIdx.x % p.slices, tile = blockIdx.x / p.slices, share = slice * 16 + w, shares = 16 * p.slices;
    const int r0 = tile / across * 32, col = tile % across * WIDE + NC * (lane & 31);
    const float* a = p.y + (int64_t)min(r0 + (lane & 31), p.M - 1) * p.Vp + 4 * hl;
    const T* b = (const T*)p.w + min(col, p.d - NC);
    const int n = p.Vp / 8, s1 = (int)((int64_t)n * (share + 1) / shares);
    constexpr int U = 4;
    for (int s = (int)((int64_t)n * share / shares); s < s1; s += U) {
      float x[U][4], y[U][4][NC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = min(s + u, s1 - 1);
        VecIO<float, 4>::load(a + 8 * at, x[u]);
#pragma unroll
        for (int t = 0; t < 4; ++t) VecIO<T, NC>::load(b + (int64_t)min(8 * at + 4 * hl + t, p.V - 1) * p.ldw, y[u][t]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t) {              // entries behind the table count as zero: y is zero there, w is not read
          const bool ok = s + u < s1 && 8 * (s + u) + 4 * hl + t < p.V;
          const float f = ok ? x[u][t] : 0.f;
#pragma unroll
          for (int k = 0; k < NC; ++k) c[k] = __builtin_amdgcn_mfma_f32_32x32x2f32(f, ok ? y[u][t][k] : 0.f, c[k], 0, 0, 0);
        }
    }
    const int row = r0 + sub;
    float s[NC];
#pragma unroll
    for (int half = 0; half < NC; ++half) {
      put(half);
      s[half] = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) s[half] += part[k][threadIdx.x];
      __syncthreads();
    }
    if (row < p.M && col < p.d) {
      const float g = p.coef[row];
      float* at = p.part + ((int64_t)slice * p.M + row) * p.d + col;
      if (p.part) {
        if (p.add) {
          float had[NC];
          VecIO<float, NC>::load(at, had);
#pragma unroll
          for (int k = 0; k < NC; ++k) s[k] += had[k];
        }
        VecIO<float, NC>::store(at, s);
      } else {
#pragma unroll
        for (int k = 0; k < NC; ++k) s[k] = g == 0.f ? 0.f : g * s[k];
        VecIO<T, NC>::store((T*)p.dh + (int64_t)row * p.ld_dh + col, s);
      }
    }
    return;
  }
  const int per = p.waves, held = 16 / per, b = blockIdx.x - p.n_dh, slice = b % p.row_slices;
  const int tiles = (p.V + 31) / 32 * across, first = b / p.row_slices * held;
  auto store = [&](int e, int col, const float (&o)[NC]) {
    if (e >= p.V || col >= p.d) return;
    if (p.part_w) VecIO<float, NC>::store(p.part_w + ((int64_t)slice * p.V + e) * p.d + col, o);
    else VecIO<T, NC>::store((T*)p.dw + (int64_t)e * p.ld_dw + col, o);
  };
  {
    const int tile = first + w / per, share = slice * per + w % per, shares = per * p.row_slices;
    if (tile < tiles) {
      const int e = tile / across * 32 + (lane & 31), col = tile % across * WIDE + NC * (lane & 31);
      const float* a = p.y + min(e, p.V - 1);
      const T* b = (const T*)p.h + min(col, p.d - NC);
      const int n = (p.M + 7) / 8, s1 = (int)((int64_t)n * (share + 1) / shares);
      constexpr int U = 2;
      for (int s = (int)((int64_t)n * share / shares); s < s1; s += U) {
        float x[U][4], y[U][4][NC], g[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int r = min(8 * (s + u) + 4 * hl + t, p.M - 1);
            x[u][t] = a[(int64_t)r * p.Vp];
            VecIO<T, NC>::load(b + (int64_t)r * p.ldh, y[u][t]);
            g[u][t] = p.coef[r];
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int t = 0; t < 4; ++t) {            // rows without a gradient count as zero, whatever they hold
            const bool ok = s + u < s1 && 8 * (s + u) + 4 * hl + t < p.M && g[u][t] != 0.f;
            const float f = ok ? x[u][t] : 0.f;
#pragma unroll
            for (int k = 0; k < NC; ++k)
              c[k] = __builtin_amdgcn_mfma_f32_32x32x2f32(f, ok ? g[u][t] * y[u][t][k] : 0.f, c[k], 0, 0, 0);
          }
      }
    }
  }
  if (per == 1) {                                  // nothing to join
    const int tile = first + w;
    if (tile >= tiles) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float o[NC];
#pragma unroll
      for (int k = 0; k < NC; ++k) o[k] = c[k][r];
      store(tile / across * 32 + 8 * (r >> 2) + 4 * hl + (r & 3), tile % across * WIDE + NC * (lane & 31), o);
    }
    return;
  }
  float s[4][NC];
#pragma unroll
  for (int half = 0; half < NC; ++half) {
    put(half);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s[q][half] = 0.f;
      if (q < held)
        for (int k = q * per; k < (q + 1) * per; ++k) s[q][half] += part[k][threadIdx.x];
    }
    __syncthreads();
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int tile = first + q;
    if (q < held && tile < tiles) store(tile / across * 32 + sub, tile % across * WIDE + NC * (lane & 31), s[q]);
  }
}

int launch_xent_direct_z(int dtype, bool grad, const XentDirect& p, hipStream_t st) {
  const int64_t blocks = (int64_t)((p.Vp + 127) / 128) * ((p.M + 31) / 32);
  NMTGAN_REQUIRE(dtype == NMTGAN_F32 || (grad && dtype == NMTGAN_BF16), "linear_xent: no direct form of dtype %d", dtype);
  NMTGAN_REQUIRE(blocks < (1LL << 31), "linear_xent: too many tiles");
  const dim3 grid((unsigned)blocks);
  if (!grad) hipLaunchKernelGGL((xent_direct_z_kernel<float, false>), grid, dim3(256), 0, st, p);
  else if (dtype == NMTGAN_F32) hipLaunchKernelGGL((xent_direct_z_kernel<float, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((xent_direct_z_kernel<bf16_t, true>), grid, dim3(256), 0, st, p);
  NMTGAN_CHECK_LAUNCH("linear_xent_direct");
  return 0;
}
int launch_xent_direct_grads(int dtype, XentDirect p, hipStream_t st) {
  const int across = (p.d + 32 * p.cols - 1) / (32 * p.cols);
  p.n_dh = (p.M + 31) / 32 * across * p.slices;
  const int64_t tiles = (int64_t)(p.V + 31) / 32 * across, held = 16 / p.waves;
  const int64_t grid = p.n_dh + (tiles + held - 1) / held * p.row_slices;
  NMTGAN_REQUIRE(grid < (1LL << 31), "linear_xent_grads: too many tiles");
  NMTGAN_REQUIRE(dtype == NMTGAN_F32 || dtype == NMTGAN_BF16, "linear_xent_grads: no direct form of dtype %d", dtype);
  auto launch = [&](auto type) {
    using T = decltype(type);
    if (p.cols == 2) hipLaunchKernelGGL((xent_direct_grads_kernel<T, 2>), dim3((unsigned)grid), dim3(1024), 0, st, p);
    else hipLaunchKernelGGL((xent_direct_grads_kernel<T, 1>), dim3((unsigned)grid), dim3(1024), 0, st, p);
  };
  if (dtype == NMTGAN_F32) launch(float{});
  else launch(bf16_t{});
  NMTGAN_CHECK_LAUNCH("linear_xent_direct_grads");
  return 0;
}

}  // namespace nmtgan
