// Products in 8-bit integers with a scale for each token and each channel (include/pie_b200.h): y[m, n] = bf16(s_m t_n sum_k c[m, k] w[n, k]).  Compiled with pie_qmm.cu,
// whose pipeline word it shares.
//
//   * int8_rows_kernel: a token's features as integers, c = x / s rounded to the nearest, s = max |x| / 127 (times the 32-bit 1 / 127); the layer's norm in front of it.
//   * more than kInt8Few rows: the GEMM core of pie_gemm.cuh on the integer tensor pipe (tcgen05 kind::i8, twice the multiply-adds of bf16 in a byte of shared memory and of
//     time), scales and residual in its epilogue.
//   * up to that: int8_few_kernel, bound by the stream of weights.
// Sums are exact (32-bit integers: K up to 131072), so it is the same result whichever way the product goes.
#pragma once
#include "pie_gemm.cuh"
#include "pie_internal.h"

namespace pie {

// ---------------------------------------------------------------------------------------------------- rows
// Eight codes: the quotients rounded by adding 1.5 2^23, whose sum has the code in its lowest byte.  A quotient by 1 / s is off by less than 2e-5: where one of the eight is as near to a half,
// all are taken by division.  (Asked of each by itself, 8191 rows of 14336 115 us.)  s < 1e-30: by division too, since 1 / s may not be a number.
__device__ __forceinline__ uint2 int8_codes(const uint4& v, float s, float inv) {
  const uint32_t q[4] = {v.x, v.y, v.z, v.w};
  float u[8], near = s < 1e-30f ? 0.f : 1.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = (e & 1 ? bf16hi(q[e >> 1]) : bf16lo(q[e >> 1])) * inv;
    u[e] = t + 12582912.f;
    near = fminf(near, fabsf(fabsf(t - (u[e] - 12582912.f)) - 0.5f));
  }
  if (near < 1e-4f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = rintf(fminf(fmaxf(__fdiv_rn(e & 1 ? bf16hi(q[e >> 1]) : bf16lo(q[e >> 1]), s), -127.f), 127.f)) + 12582912.f;
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = __byte_perm(__byte_perm(__float_as_uint(u[4 * h]), __float_as_uint(u[4 * h + 1]), 0x0040), __byte_perm(__float_as_uint(u[4 * h + 2]), __float_as_uint(u[4 * h + 3]), 0x0040), 0x5410);
  return make_uint2(w[0], w[1]);
}
// eight features through the norm, rounded as pie_rms_norm rounds
__device__ __forceinline__ uint4 int8_norm(const uint4& v, const uint4& g, float inv) {
  const uint32_t q[4] = {v.x, v.y, v.z, v.w}, w[4] = {g.x, g.y, g.z, g.w};
  uint32_t r[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t n = pack_bf16(bf16lo(q[e]) * inv, bf16hi(q[e]) * inv);
    r[e] = pack_bf16(bf16lo(n) * bf16lo(w[e]), bf16hi(n) * bf16hi(w[e]));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ float int8_squares(const uint4& v, float ss) {
  const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) { ss = fmaf(bf16lo(q[e]), bf16lo(q[e]), ss); ss = fmaf(bf16hi(q[e]), bf16hi(q[e]), ss); }
  return ss;
}
__device__ __forceinline__ uint32_t int8_most(const uint4& v, uint32_t m) {   // of two halves each: magnitudes in the order of their bits
  constexpr uint32_t ABS = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(__vmaxu2(m, v.x & ABS), __vmaxu2(v.y & ABS, v.z & ABS)), v.w & ABS);
}

// A CTA of THREADS a row.  NV 16-byte pieces a thread are held in registers, so that a row is read once; NV 0: rows of any length, read again for each of the passes.  (Four pieces and a norm: four CTAs
// an SM, which takes 64 registers; left to itself 68, and 8191 rows of 8192 70.5 us in place of 63.8.)
template <int NV, int THREADS, bool NORM>
__global__ void __launch_bounds__(THREADS, NORM && THREADS == 256 && NV == 4 ? 4 : 0) int8_rows_kernel(int8_t* codes, float* scales, const uint16_t* x, long long x_ld, const uint16_t* norm, float eps, int nvec) {
  constexpr int WARPS = THREADS / 32;
  __shared__ float sums[8];
  __shared__ uint32_t most[WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint4* const xr = reinterpret_cast<const uint4*>(x + blockIdx.x * x_ld);
  const uint4* const wr = reinterpret_cast<const uint4*>(norm);
  uint2* const out = reinterpret_cast<uint2*>(codes) + (size_t)blockIdx.x * nvec;
  uint4 v[NV ? NV : 1], g[NV ? NV : 1];
  if (NV) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = tid + THREADS * j;
      v[j] = i < nvec ? xr[i] : make_uint4(0, 0, 0, 0);
      if (NORM) g[j] = i < nvec ? __ldg(wr + i) : make_uint4(0, 0, 0, 0);
    }
  }
  float inv_rms = 0.f;
  if (NORM) {
    // A row's bits do not depend on how many rows come with it: 256 threads and 1024 add the squares up in one order, of pieces 1024 apart, then of four such sums 256 apart, then of 32 lanes.
    // (As 1024 threads would by themselves, lanes first, it takes 256 threads four turns among their lanes: 8191 rows of 8192 75.9 us; so 63.8.)
    constexpr int SUMS = THREADS == 256 && NV != 1 && NV != 2 ? 4 : 1;
    float part[SUMS] = {};
    if (NV) {
#pragma unroll
      for (int j = 0; j < NV; ++j) part[j % SUMS] = int8_squares(v[j], part[j % SUMS]);
    } else {
      for (int i = tid; i < nvec; i += THREADS * SUMS)
#pragma unroll
        for (int c = 0; c < SUMS; ++c)
          if (i + THREADS * c < nvec) part[c] = int8_squares(xr[i + THREADS * c], part[c]);
    }
    float ss;
    if (THREADS == 1024) {
      __shared__ float parts[THREADS];
      parts[tid] = part[0];
      __syncthreads();
      if (warp < 8) ss = (parts[tid] + parts[tid + 256]) + (parts[tid + 512] + parts[tid + 768]);
    } else {
      ss = SUMS == 4 ? (part[0] + part[SUMS == 4 ? 1 : 0]) + (part[SUMS == 4 ? 2 : 0] + part[SUMS == 4 ? 3 : 0]) : part[0];
    }
    if (warp < 8) {
      ss = warp_sum(ss);
      if (lane == 0) sums[warp] = ss;
    }
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += sums[w];
    inv_rms = 1.0f / sqrtf(total / (float)(nvec * 8) + eps);
  }
  uint32_t m = 0;
  if (NV) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (NORM) v[j] = int8_norm(v[j], g[j], inv_rms);
      m = int8_most(v[j], m);   // (a piece behind the row's end is zeros, or 0 * inv_rms: where that is not 0, the row has no finite norm)
    }
  } else {
    for (int i = tid; i < nvec; i += THREADS) {
      const uint4 a = xr[i];
      m = int8_most(NORM ? int8_norm(a, __ldg(wr + i), inv_rms) : a, m);
    }
  }
  m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
  if (lane == 0) most[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; ++w) m = max(m, most[w]);
  // an infinity or a NaN: nothing of the row has a value, and its products are NaN
  const float amax = __uint_as_float(m << 16), s = m < 0x7f80u ? amax * (1.f / 127.f) : __uint_as_float(0x7fc00000u);
  if (tid == 0) scales[blockIdx.x] = s;
  const bool some = s > 0.f;
  const float inv = some && s >= 1e-30f ? __fdiv_rn(1.f, s) : 0.f;
  auto put = [&](int i, const uint4& a) {
    if (i >= nvec) return;
    out[i] = some ? int8_codes(a, s, inv) : make_uint2(0, 0);
  };
  if (NV) {
#pragma unroll
    for (int j = 0; j < NV; ++j) put(tid + THREADS * j, v[j]);
  } else {
    for (int i = tid; i < nvec; i += THREADS) {
      const uint4 a = xr[i];
      put(i, NORM ? int8_norm(a, __ldg(wr + i), inv_rms) : a);
    }
  }
}

template <int THREADS, bool NORM>
static cudaError_t launch_int8_rows_by(int8_t* codes, float* scales, const uint16_t* x, long long x_ld, int rows, int nvec, const uint16_t* norm, float eps, cudaStream_t st) {
  const int per = (nvec + THREADS - 1) / THREADS;
  auto kern = per <= 1 ? int8_rows_kernel<1, THREADS, NORM> : per <= 2 ? int8_rows_kernel<2, THREADS, NORM> : per <= 4 ? int8_rows_kernel<4, THREADS, NORM>
              : per <= 8 && THREADS < 1024 ? int8_rows_kernel<THREADS < 1024 ? 8 : 4, THREADS, NORM> : int8_rows_kernel<0, THREADS, NORM>;
  count_launch();
  return launch_pdl(kern, dim3((unsigned)rows), dim3(THREADS), 0, st, codes, scales, x, x_ld, norm, eps, nvec);
}
// Few rows are a chain (loads, largest, division, codes) that the product waits for: as many threads as a row has pieces, up to 1024 (a row of 14336 as 256 threads 6.6 us); many rows are bound by
// HBM (8191 of 14336 81.8 us at 127 registers, of which the norm's weights were 32).
cudaError_t launch_int8_rows(int8_t* codes, float* scales, const uint16_t* x, long long x_ld, int rows, int K, const uint16_t* norm, float eps, cudaStream_t st) {
  const int nvec = K / 8;
  if (rows <= num_sms() && nvec > 512)
    return norm ? launch_int8_rows_by<1024, true>(codes, scales, x, x_ld, rows, nvec, norm, eps, st) : launch_int8_rows_by<1024, false>(codes, scales, x, x_ld, rows, nvec, norm, eps, st);
  return norm ? launch_int8_rows_by<256, true>(codes, scales, x, x_ld, rows, nvec, norm, eps, st) : launch_int8_rows_by<256, false>(codes, scales, x, x_ld, rows, nvec, norm, eps, st);
}

// ---------------------------------------------------------------------------------------------------- many rows
// y = bf16(sum s_m t_n), and a residual added to that as pie_add adds it
struct Int8Store {
  static constexpr bool INTEGER = true;
  uint16_t* y;
  const uint16_t* residual;
  const float *sx, *sw;
  int M, N;
  __device__ __forceinline__ void operator()(int, int row0, int col, const uint32_t (&v)[32], uint32_t buf, int lane) const {
    if (row0 >= M || col >= N) return;
    const float s = row0 + lane < M ? __ldg(sx + row0 + lane) : 0.f;
    float t[32];
    if (col + 32 <= N) {
#pragma unroll
      for (int q = 0; q < 8; ++q) *reinterpret_cast<float4*>(t + 4 * q) = __ldg(reinterpret_cast<const float4*>(sw + col) + q);
    } else {
      const float mine = col + lane < N ? __ldg(sw + col + lane) : 0.f;
#pragma unroll
      for (int q = 0; q < 32; ++q) t[q] = __shfl_sync(0xffffffffu, mine, q);
    }
    auto value = [&](int q) { return (float)(int)v[q] * s * t[q]; };
    const size_t first = (size_t)row0 * N + col;
    if ((N & 7) == 0) {   // as QmmStore
      auto at = [&](int r, int c) { return buf + r * 64 + ((c ^ ((r >> 1) & 3)) << 4); };
#pragma unroll
      for (int c = 0; c < 4; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at(lane, c)), "r"(pack_bf16(value(8 * c), value(8 * c + 1))),
                     "r"(pack_bf16(value(8 * c + 2), value(8 * c + 3))), "r"(pack_bf16(value(8 * c + 4), value(8 * c + 5))),
                     "r"(pack_bf16(value(8 * c + 6), value(8 * c + 7))) : "memory");
      const int c = lane & 3;
      uint4 res[4];
      if (residual) {   // (may lie where y goes: a thread reads what it writes)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + (lane >> 2);
          res[i] = make_uint4(0, 0, 0, 0);
          if (row0 + r < M && col + 8 * c < N) res[i] = *reinterpret_cast<const uint4*>(residual + first + (size_t)r * N + 8 * c);
        }
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        uint4 o = lds128(at(r, c));
        if (residual) { o.x = sum(o.x, res[i].x); o.y = sum(o.y, res[i].y); o.z = sum(o.z, res[i].z); o.w = sum(o.w, res[i].w); }
        if (row0 + r < M && col + 8 * c < N) *reinterpret_cast<uint4*>(y + first + (size_t)r * N + 8 * c) = o;
      }
      __syncwarp();
    } else if (row0 + lane < M) {
#pragma unroll
      for (int q = 0; q < 32; ++q)
        if (col + q < N) {
          const size_t p = first + (size_t)lane * N + q;
          const uint16_t o = f2bf(value(q));
          y[p] = residual ? f2bf(bf16lo(o) + bf16lo(residual[p])) : o;
        }
    }
  }
  static __device__ __forceinline__ uint32_t sum(uint32_t a, uint32_t b) { return pack_bf16(bf16lo(a) + bf16lo(b), bf16hi(a) + bf16hi(b)); }
};

// x and w as the core counts them: rows of K / 2 pairs of integers, K steps of 64 pairs
static cudaError_t launch_int8_core(const Int8Store& epi, const int8_t* codes, const int8_t* w, int K, cudaStream_t st) {
  const int sms = num_sms();
  GemmArgs a = {};
  a.M = epi.M; a.N = epi.N; a.K = (K + 127) / 128 * 64; a.nb = 1;
  const GemmChoice c = gemm_choose(a.M, a.N, a.K, 1, sms, false);
  a.mt = c.mt; a.nt = c.nt; a.k_per = c.k_per; a.group_m = 8;
  CUtensorMap mx, mw;
  if (!gemm_map(&mx, codes, 2, K / 2, a.M, K, 1, 0, 128) || !gemm_map(&mw, w, 2, K / 2, a.N, K, 1, 0, c.pair ? c.bn / 2 : c.bn)) return cudaErrorNotSupported;
  count_launch();
  if (!c.pair)
    return c.ranks == 1 ? gemm_launch<1, 128, 0, false>(mx, mw, a, epi, 1, sms, st) : gemm_launch<1, 128, 0, true>(mx, mw, a, epi, c.ranks, sms, st);
  if (c.bn == 256) return gemm_launch<2, 256, 0, false>(mx, mw, a, epi, 1, sms, st);
  return c.bn == 192 ? gemm_launch<2, 192, 0, false>(mx, mw, a, epi, 1, sms, st) : gemm_launch<2, 128, 0, false>(mx, mw, a, epi, 1, sms, st);
}

// ---------------------------------------------------------------------------------------------------- few rows
// What bounds it is the stream of weights, so the shape follows from keeping that going on every SM:
//   * the weights are the MMA's A operand, 128 channels a tile, and the rows, padded to 16, its N: tcgen05.mma kind::i8, M128 N16 K32.
//   * the tiles' K steps of 128 bytes lie one behind the other on a line and every CTA has the same length of it, so that no SM waits for others' tiles.  A CTA's TMA ring
//     goes on from one tile to the next; two accumulators, so that a tile's end is under the next one's start.
//   * a tile that lies in several shares is added up in 32-bit integers: every CTA adds its part to the tile's sums in the workspace, and the last one to come takes them
//     and leaves zeros.  (Integers: the same sum in any order.)
// us, codes given, weights not in L2; this and the core: 1 row 6144 x 4096 9.0, 11; 4096 x 14336 14.2, 17.0; 28672 x 4096 22.7, 25.5 (5.2 TB/s).  16 rows 10.6, 15.7, 24.7.  What does not
// shrink with the weights, some 5 us, is the start, sums and counter in L2, and their way back.  32 rows (as wider MMAs) 14.0, 18.4, 28.6: that many sums are sooner added up in the
// shared memory of the core's clusters (11.0, 17.0, 25.6).
constexpr int kInt8Few = 16;   // rows, at most
constexpr int kInt8Ahead = 26; // K steps of 16 KB a CTA asks L2 for
struct Int8Few {
  static constexpr int A_STAGE = 128 * 128, B_STAGE = kInt8Few * 128, S = 11;
  static constexpr int SMEM = 1024 + S * (A_STAGE + B_STAGE);
  static constexpr int THREADS = 192, W_TMA = 4, W_MMA = 5;
  static constexpr int TMEM_COLS = 2 * kInt8Few;
  static_assert(SMEM <= 226 * 1024, "shared memory");
};
struct Int8FewArgs {
  uint16_t* y;
  const uint16_t* residual;
  const float *sx, *sw;
  int M, N, nk, ctas;        // nk: K steps of a tile
  long long steps;           // of all tiles
  int* sums;                 // [tiles][16][128], zero between launches
  unsigned int* count;       // [tiles], zero between launches
};

__global__ void __launch_bounds__(Int8Few::THREADS, 1)
int8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Int8FewArgs a) {
  using T = Int8Few;
  constexpr int S = T::S, NB = kInt8Few;
  constexpr uint32_t IDESC = umma_idesc_i8<128, NB>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], tfull_bar[2], tempty_bar[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, last_flag;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u, smA = base, smB = base + S * T::A_STAGE;
  // this CTA's part of the line
  const long long lo = (long long)blockIdx.x * a.steps / a.ctas, hi = (long long)(blockIdx.x + 1) * a.steps / a.ctas;
  const int tile0 = (int)(lo / a.nk), k_first = (int)(lo - (long long)tile0 * a.nk), total = (int)(hi - lo);
  if (tid == 0) {
    for (int s = 0; s < S; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&tfull_bar[b], 1); mbar_init(&tempty_bar[b], 4); }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == T::W_MMA) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(T::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == T::W_TMA && lane == 0) {
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    // The first weights on their way to L2 while the launch before this one, which makes the codes, goes on (nothing is read ahead of the wait: it may have written them): as much as
    // half of L2 holds.
    for (int i = 0; i < min(kInt8Ahead, total); ++i) {
      const int kb = (k_first + i) % a.nk, t = tile0 + (k_first + i) / a.nk;
      gemm_prefetch_3d(&map_w, kb * 64, t * 128, 0);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  volatile int* const abortp = &abort_flag;
  pdl_launch_dependents();
  pdl_wait();

  if (warp < 4) {
    // ---------------------------------------------------------------- a channel a thread
    // A warp whose wait ran out has no sums to give, but walks on: its CTA's barriers count it, and each part of a tile is counted and each tile's sums are cleared all the same, so that
    // the workspace is left at zero.
    bool alive = true;
    int done = 0;
    for (int t = tile0, k0 = k_first, i = 0; done < total; ++t, k0 = 0, ++i) {
      const int n = min(a.nk - k0, total - done), b = i & 1;
      done += n;
      alive = alive && gemm_wait_warp(smem_u32(&tfull_bar[b]), (i >> 1) & 1, abortp);
      const bool whole = n == a.nk;
      const int channel = t * 128 + tid;
      const bool there = channel < a.N;
      const float tw = there ? __ldg(a.sw + channel) : 0.f;
      int* const sums = a.sums + (size_t)t * NB * 128 + tid;
      auto put = [&](int m, int sum) {
        const size_t p = (size_t)m * a.N + channel;
        const uint16_t o = f2bf((float)sum * __ldg(a.sx + m) * tw);
        a.y[p] = a.residual ? f2bf(bf16lo(o) + bf16lo(a.residual[p])) : o;
      };
      if (alive) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t v[16];
        tmem_ld16(tmem + (uint32_t)(b * NB) + ((uint32_t)(warp * 32) << 16), v);
        tmem_ld_wait();
#pragma unroll
        for (int q = 0; q < 16; ++q)
          if (q < a.M && there) {
            if (whole) put(q, (int)v[q]);
            else atomicAdd(sums + q * 128, (int)v[q]);
          }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (alive && lane == 0) mbar_arrive(&tempty_bar[b]);
      if (!whole) {
        // the CTAs whose shares the tile lies in: that of its first step, to that of its last
        const long long s0 = (long long)t * a.nk, s1 = s0 + a.nk - 1;
        const unsigned parts = (unsigned)(((s1 + 1) * a.ctas - 1) / a.steps - ((s0 + 1) * a.ctas - 1) / a.steps + 1);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (tid == 0) {
          unsigned int before;   // (release and acquire reach, through the barriers, what every warp added and will read)
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.count + t) : "memory");
          last_flag = before == parts - 1;
          if (last_flag) a.count[t] = 0;   // for the next launch: nobody else comes
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (last_flag && there) {
#pragma unroll 1
          for (int c = 0; c < a.M; c += 8) {
            int v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = c + q < a.M ? __ldcg(sums + (c + q) * 128) : 0;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (c + q < a.M) {
                __stcg(sums + (c + q) * 128, 0);
                put(c + q, v[q]);
              }
          }
        }
      }
    }
  } else if (warp == T::W_TMA) {
    if (lane == 0) {
      int t = tile0, kb = k_first;
      for (int it = 0; it < total; ++it) {
        const int s = it % S;
        if (!gemm_wait(smem_u32(&empty_bar[s]), ((it / S) & 1) ^ 1, abortp)) break;
        mbar_arrive_expect_tx(&full_bar[s], T::A_STAGE + T::B_STAGE);
        gemm_tma_3d<1>(smA + s * T::A_STAGE, &map_w, smem_u32(&full_bar[s]), kb * 64, t * 128, 0);
        gemm_tma_3d<1>(smB + s * T::B_STAGE, &map_x, smem_u32(&full_bar[s]), kb * 64, 0, 0);
        if (++kb == a.nk) { kb = 0; ++t; }
      }
    }
  } else {
    const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t da0 = umma_desc_sw128(smA), db0 = umma_desc_sw128(smB);
    bool alive = true;   // a lane's own: a wait that expires only keeps the elected lane from issuing
    int it = 0;
    for (int k0 = k_first, i = 0; it < total; k0 = 0, ++i) {
      const int n = min(a.nk - k0, total - it), b = i & 1;
      alive &= gemm_wait(smem_u32(&tempty_bar[b]), ((i >> 1) & 1) ^ 1, abortp);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (int j = 0; j < n; ++j, ++it) {
        const int s = it % S;
        alive &= gemm_wait(smem_u32(&full_bar[s]), (it / S) & 1, abortp);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_one() && alive) {
          const uint64_t da = da0 + (uint64_t)(s * (T::A_STAGE >> 4)), db = db0 + (uint64_t)(s * (T::B_STAGE >> 4));
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) gemm_mma<1, true>(acc + b * NB, da + 2 * k4, db + 2 * k4, IDESC, (j > 0 || k4 > 0) ? 1u : 0u);
          gemm_commit<1>(smem_u32(&empty_bar[s]));
          if (j == n - 1) gemm_commit<1>(smem_u32(&tfull_bar[b]));
        }
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abortp) gemm_drain();
  if (warp == T::W_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(T::TMEM_COLS) : "memory");
}

static cudaError_t launch_int8_few(Int8FewArgs a, const int8_t* codes, const int8_t* w, int K, cudaStream_t st) {
  using T = Int8Few;
  static std::atomic<unsigned long long> served{0};
  const cudaError_t set = once_per_device(served, [] { return cudaFuncSetAttribute(int8_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM); });
  if (set != cudaSuccess) return set;
  CUtensorMap mw, mx;
  if (!gemm_map(&mw, w, 2, K / 2, a.N, K, 1, 0, 128) || !gemm_map(&mx, codes, 2, K / 2, a.M, K, 1, 0, kInt8Few)) return cudaErrorNotSupported;
  const int tiles = (a.N + 127) / 128, sms = num_sms();
  a.nk = (K + 127) / 128;
  a.steps = (long long)tiles * a.nk;
  a.ctas = (int)(a.steps < sms ? a.steps : sms);
  count_launch();
  return launch_pdl(int8_few_kernel, dim3((unsigned)a.ctas), dim3(T::THREADS), T::SMEM, st, mw, mx, a);
}

size_t int8_workspace_bytes(int M, int N) {
  if (M > kInt8Few) return 0;
  const size_t tiles = ((size_t)N + 127) / 128;
  return (tiles * 4 + 255) / 256 * 256 + tiles * 128 * kInt8Few * 4;
}

cudaError_t launch_int8_matmul(uint16_t* y, const int8_t* codes, const float* sx, const int8_t* w, const float* sw, const uint16_t* residual, int M, int N, int K, void* ws,
                               cudaStream_t st) {
  if (M > kInt8Few) return launch_int8_core(Int8Store{y, residual, sx, sw, M, N}, codes, w, K, st);
  const size_t tiles = ((size_t)N + 127) / 128;
  Int8FewArgs a = {};
  a.y = y; a.residual = residual; a.sx = sx; a.sw = sw; a.M = M; a.N = N;
  a.count = (unsigned int*)ws;
  a.sums = (int*)((uint8_t*)ws + (tiles * 4 + 255) / 256 * 256);
  return launch_int8_few(a, codes, w, K, st);
}

}  // namespace pie
