// Causal attention of every request's new tokens over its pages (include/pie_b200.h), on the 5th-generation tensor cores.  Compiled with pie_fa_prefill.cu, whose
// tile this is (two softmax groups of four warps, a TMA warp, a warp that issues the MMAs) and whose pipeline word it shares.
//
// Replaces, for the rows of a ragged step, mx.fast.scaled_dot_product_attention with the causal mask of create_attention_mask (PIE/models/base.py:18-53, 92-113).
//
// The rows of a query tile are the query heads of one key / value head, token by token (32 tokens of 4 heads): keys and values are read once for all of them, and a tile
// of few tokens crosses the diagonal in few key tiles.  An item (pie_step_plan.h) has either
//   * rows in both query tiles: they walk the same key tiles, one tile's softmax under the other's MMAs, as in the prompt's kernel -- bound by softmax and tensor pipe; or
//   * one query tile, of a few tokens as a rule: the groups take every other key tile of it, each with its own maximum, sum and accumulator, which meet at the end through
//     tensor memory (the groups' warps read the same lanes) -- bound by the stream of keys and values.  Rows without a token cost no exponentials.
// A CTA per SM walks the pieces that the plan dealt out to it.  A piece of a cut item leaves its maxima, sums and unnormalised results (fp32) in its CTA's place of the
// workspace, and the last CTA of the item to arrive adds all pieces up in their order: the same bits whichever that is.
// Keys that a row must not see get weight 0; values behind the item's last key are cleared in shared memory, since 0 * NaN is not 0.
// Every wait is bounded (pie_gemm.cuh); a warp whose wait ran out does nothing more, but walks on through the barriers of the eight softmax warps.
#include "pie_step_plan.h"

namespace pie {

struct ChunkArgs {
  uint16_t* out;
  int Hq, G, tile_tokens;      // G: query heads of a key / value head
  int rows, requests;
  float scale_log2e;
  const int32_t *ranges, *table, *row_starts;
  const StepPiece* pieces;
  int blocks;
  unsigned int* count;         // [kStepMaxCtas], zero between launches
  float* part;                 // [2 CTAs][D / 4][256][4] results, [256][2] maxima and sums
  int rest;
};
template <int D>
constexpr int kChunkRecord = 256 * D + 512;   // floats

// a piece as the roles walk it
struct ChunkPiece {
  int row0, pos0, tokens, request, head, k0, n, first, pieces;
  bool pair;
  int cnt0, cnt1;              // key tiles of either group
  __device__ __forceinline__ int cnt(int g) const { return g ? cnt1 : cnt0; }
};
__device__ __forceinline__ bool chunk_piece(const ChunkArgs& a, int& at, int end, ChunkPiece& p) {
  while (at < end) {
    const int4* const e = reinterpret_cast<const int4*>(a.pieces + at++);
    const int4 x = __ldg(e), y = __ldg(e + 1), z = __ldg(e + 2);
    p.row0 = x.x; p.pos0 = x.y; p.tokens = x.z; p.request = x.w;
    p.head = y.x; p.k0 = y.y; p.n = y.z - y.y; p.first = y.w;
    p.pieces = z.x;
    if (p.n <= 0) continue;
    p.pair = p.tokens > a.tile_tokens;
    if (p.pair) {
      p.cnt0 = max(0, min(p.n, (p.pos0 + a.tile_tokens - 1) / kStepTile + 1 - p.k0));
      p.cnt1 = p.n;
    } else {
      p.cnt0 = (p.n + 1) / 2;
      p.cnt1 = p.n / 2;
    }
    return true;
  }
  p.n = p.cnt0 = p.cnt1 = 0;
  return false;
}
__device__ __forceinline__ void chunk_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }   // the eight softmax warps

template <int D>
__global__ void __launch_bounds__(FapTile<D>::THREADS, 1)
chunk_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ ChunkArgs a) {
  using T = FapTile<D>;
  constexpr uint32_t ID_S = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t ID_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
  constexpr int COL_S = 0, COL_O = 256;   // + g * 128, + g * D
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
  __shared__ float2 ml[2][128];           // a row's maximum and sum: of the two groups of a tile, of the rows of a cut item
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, last_flag;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t smQ = base, smK = base + 2 * T::TILE, smV = base + 4 * T::TILE;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1);
      mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 8 && lane < 3) tma_prefetch_desc(lane == 0 ? &map_q : lane == 1 ? &map_k : &map_v);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  volatile int* const abortp = &abort_flag;
  pdl_launch_dependents();
  pdl_wait();   // (the set-up above ran under the end of the launch before this one)
  const int begin = __ldg(a.ranges + 2 * blockIdx.x), end = __ldg(a.ranges + 2 * blockIdx.x + 1);

  // All barriers are counted over the CTA's pieces: a role keeps the number of key tiles (of its group, of K and V) before its piece.
  // Registers as in the prompt's kernel: 8 x 32 x 216 + 4 x 32 x 64 = 63488 of the 384 x 168 = 64512 at launch.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------------------------------------------ softmax of group g
    const int g = warp >> 2, quad = warp & 3, r = quad * 32 + lane, tok = r / a.G, hq = r - tok * a.G;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t tS = tmem + COL_S + g * 128 + lanes, tO = tmem + COL_O + lanes;
    int c[2] = {0, 0}, cv = 0;     // key tiles of either group, tiles of V, before this piece
    bool alive = true;
    int at = begin;
    ChunkPiece p, next;
    bool more = chunk_piece(a, at, end, next);
    while (more) {
      p = next;
      more = chunk_piece(a, at, end, next);
      const int t0 = p.pair ? g * a.tile_tokens : 0;                      // the tile's first token of the item
      const bool live = tok < a.tile_tokens && t0 + tok < p.tokens;
      const bool busy = __any_sync(0xffffffffu, live);
      const int lim = p.pos0 + t0 + tok, first_lim = __shfl_sync(0xffffffffu, lim, 0);   // last key this row, the warp's first row sees
      const int keys = p.pos0 + p.tokens, tail = keys & 127, cnt = p.cnt(g);
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < cnt; ++i) {
        const int step = p.pair ? i : 2 * i + g, j = p.k0 + step;
        alive = alive && gemm_wait_warp(smem_u32(&s_full[g]), (c[g] + i) & 1, abortp);
        if (!alive) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (busy) {
          float s[128];
#pragma unroll
          for (int q = 0; q < 4; ++q) fap_tmem_ld(tS + 32 * q, s + 32 * q);
          tmem_ld_wait();
          if (j * 128 + 127 > first_lim) {   // a key of this tile lies beyond some row of the warp
            const int last = lim - j * 128;
#pragma unroll
            for (int k = 0; k < 128; ++k)
              if (k > last) s[k] = -INFINITY;
          }
          float x0 = s[0], x1 = s[1], x2 = s[2], x3 = s[3];
#pragma unroll
          for (int k = 4; k < 128; k += 4) {
            x0 = fmaxf(x0, s[k]); x1 = fmaxf(x1, s[k + 1]); x2 = fmaxf(x2, s[k + 2]); x3 = fmaxf(x3, s[k + 3]);
          }
          const float mx = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * a.scale_log2e;   // (the scale is positive)
          const bool move = mx > m + 8.f;
          if (i == 0) {
            m = mx;
          } else if (__any_sync(0xffffffffu, move)) {
            const float f = move ? fap_exp2(m - mx) : 1.f;   // m == -inf: 0, and everything it multiplies is 0
            if (move) m = mx;
            l *= f;
            // O holds the tiles before this one once their product has finished
            alive = gemm_wait_warp(smem_u32(&o_full[g]), (c[g] + i - 1) & 1, abortp);
            if (!alive) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              float o[32];
              fap_tmem_ld(tO + g * D + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= f;
              tmem_st32(tO + g * D + c0, reinterpret_cast<uint32_t*>(o));
            }
            tmem_st_wait();
          }
          const float ms = m == -INFINITY ? 0.f : m;
          const f32x2 sc2 = f2_pack(a.scale_log2e, a.scale_log2e), ms2 = f2_pack(-ms, -ms);
          f32x2 l01 = f2_pack(0.f, 0.f), l23 = l01;
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t w[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const f32x2 x = f2_fma(f2_pack(s[64 * hf + 2 * k], s[64 * hf + 2 * k + 1]), sc2, ms2);
              float e0, e1;
              if (k % 4 == 3) {        // every fourth pair off the approximation unit, which would otherwise bound the tile
                fap_exp2_poly(x, e0, e1);
              } else {
                float y0, y1;
                f2_unpack(x, y0, y1);
                e0 = fap_exp2(y0);
                e1 = fap_exp2(y1);
              }
              w[k] = pack_bf16(e0, e1);
              if (k & 1) l23 = f2_add(l23, f2_pack(e0, e1));
              else l01 = f2_add(l01, f2_pack(e0, e1));
            }
            tmem_st32(tS + 32 * hf, w);
          }
          float l0, l1;
          f2_unpack(f2_add(l01, l23), l0, l1);
          l += l0 + l1;
          tmem_st_wait();
        }
        if (tail && j == (keys - 1) / 128) {   // what lies behind the item's last key may be anything
          const int v = cv + step;
          alive = gemm_wait_warp(smem_u32(&v_full[v & 1]), (v >> 1) & 1, abortp);
          if (!alive) break;
          if (r >= tail)
#pragma unroll
            for (int q = 0; q < 8 * T::CH; ++q)
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(smV + (v & 1) * T::TILE + (q >> 3) * 16384 + r * 128 + (q & 7) * 16),
                           "r"(0) : "memory");
          fence_proxy_async();
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
      }
      c[0] += p.cnt0; c[1] += p.cnt1; cv += p.n;

      // ---- results.  O is read before this warp says that the next piece's first P is there, which its first product, overwriting O, waits for.
      if (p.pair) {
        if (cnt > 0) alive = alive && gemm_wait_warp(smem_u32(&o_full[g]), (c[g] - 1) & 1, abortp);
      } else {
        ml[g][r] = make_float2(m, l);
        alive = alive && gemm_wait_warp(smem_u32(&o_full[0]), (c[0] - 1) & 1, abortp);
        if (p.cnt1 > 0) alive = alive && gemm_wait_warp(smem_u32(&o_full[1]), (c[1] - 1) & 1, abortp);
        chunk_sync();
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float f0 = 1.f, f1 = 0.f;   // factors of the two accumulators of one tile
      if (!p.pair) {
        const float2 u = ml[g ^ 1][r];
        const float mx = fmaxf(m, u.x), fm = m == -INFINITY ? 0.f : fap_exp2(m - mx), fu = u.x == -INFINITY ? 0.f : fap_exp2(u.x - mx);
        l = (l == 0.f ? 0.f : l * fm) + (u.y == 0.f ? 0.f : u.y * fu);
        m = mx;
        f0 = g ? fu : fm;
        f1 = g ? fm : fu;
      }
      // columns of this group: its own accumulator, or half of both of one tile's
      const int col0 = p.pair ? 0 : g * (D / 2), col1 = p.pair ? D : col0 + D / 2;
      const uint32_t from = p.pair ? tO + g * D : tO;
      const bool two = !p.pair && p.cnt1 > 0;
      const bool whole = p.pieces == 1;
      const int rr = (p.pair ? g * 128 : 0) + r;
      float* const rec = a.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == p.first)) * kChunkRecord<D>;
      if (alive && busy && cnt + (p.pair ? 0 : 1) > 0) {
        const float inv = whole ? 1.f / l : 1.f;
        uint16_t* const o_row = a.out + ((size_t)(p.row0 + t0 + tok) * a.Hq + p.head * a.G + hq) * D;
#pragma unroll 1
        for (int c0 = col0; c0 < col1; c0 += 32) {
          float o[32];
          fap_tmem_ld(from + c0, o);
          tmem_ld_wait();
          if (two) {
            float u[32];
            fap_tmem_ld(from + D + c0, u);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = o[k] * f0 + u[k] * f1;
          }
          if (live) {
            if (whole) {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint4*>(o_row + c0 + 8 * q) =
                    make_uint4(pack_bf16(o[8 * q] * inv, o[8 * q + 1] * inv), pack_bf16(o[8 * q + 2] * inv, o[8 * q + 3] * inv),
                               pack_bf16(o[8 * q + 4] * inv, o[8 * q + 5] * inv), pack_bf16(o[8 * q + 6] * inv, o[8 * q + 7] * inv));
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                __stcg(reinterpret_cast<float4*>(rec + ((size_t)(c0 / 4 + q) * 256 + rr) * 4), make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]));
            }
          }
        }
      }
      if (!whole) {
        if (live && (p.pair || g == 0)) __stcg(reinterpret_cast<float2*>(rec + 256 * D + 2 * rr), make_float2(m, l));
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        chunk_sync();
        if (tid == 0) {
          unsigned int before;   // (release and acquire reach, through the barriers, what every warp stored and will read)
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.count + p.first) : "memory");
          last_flag = before == (unsigned)p.pieces - 1;
          if (last_flag) a.count[p.first] = 0;   // for the next launch: nobody else comes
        }
        chunk_sync();
        if (last_flag) {
          // the item's pieces: the one that opens it, and the ones of the CTAs behind, in order.  A thread a row for the sums, then four features of a row.
          const float* const rec0 = a.part + (size_t)(2 * p.first + 1) * kChunkRecord<D>;
          const size_t hop = 2 * (size_t)kChunkRecord<D>;
          auto piece = [&](int i) { return i == 0 ? rec0 : rec0 + i * hop - kChunkRecord<D>; };
          const int live_rows = p.tokens * a.G;
          auto place = [&](int e) {   // of live row e in a record
            const int t = e / a.G, tile = t / a.tile_tokens;
            return tile * 128 + e - tile * a.tile_tokens * a.G;
          };
          float2* const sums = &ml[0][0];
          if (tid < live_rows) {
            const int at_row = 256 * D + 2 * place(tid);
            float mx = -INFINITY, ls = 0.f;
#pragma unroll 4
            for (int i = 0; i < p.pieces; ++i) mx = fmaxf(mx, __ldcg(piece(i) + at_row));
#pragma unroll 4
            for (int i = 0; i < p.pieces; ++i) {
              const float2 v = __ldcg(reinterpret_cast<const float2*>(piece(i) + at_row));
              ls += v.x == -INFINITY && mx != -INFINITY ? 0.f : v.y * exp2f(v.x - mx);
            }
            sums[tid] = make_float2(mx, 1.f / ls);
          }
          chunk_sync();
          for (int e = tid; e < live_rows * (D / 4); e += 256) {
            const int c4 = e / live_rows, row = e - c4 * live_rows, q = place(row), t = row / a.G;
            const float2 s = sums[row];
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int i = 0; i < p.pieces; ++i) {
              const float mi = __ldcg(piece(i) + 256 * D + 2 * q);
              const float4 v = __ldcg(reinterpret_cast<const float4*>(piece(i) + ((size_t)c4 * 256 + q) * 4));
              if (mi == -INFINITY && s.x != -INFINITY) continue;   // (a piece without a key for this row may not have written results)
              const float f = exp2f(mi - s.x) * s.y;
              o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
            }
            *reinterpret_cast<uint2*>(a.out + ((size_t)(p.row0 + t) * a.Hq + p.head * a.G + row - t * a.G) * D + 4 * c4) =
                make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
          }
          chunk_sync();   // (the sums are read before they are written again)
        }
      } else if (!p.pair) {
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        chunk_sync();     // both groups have read both accumulators
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ------------------------------------------------------------------------------------------------ TMA
    if (warp == 8) {
      bool alive = true;
      int cq[2] = {0, 0}, ck = 0;   // pieces with a query tile g, key tiles, before this piece
      int at = begin;
      ChunkPiece p;
      while (alive && chunk_piece(a, at, end, p)) {
        const int32_t* const pages = a.table + (size_t)p.request * a.blocks;
        const int last_page = (p.pos0 + p.tokens - 1) / kStepPage;
        int first = 2 * p.k0, ids = __ldg(pages + min(first + lane, last_page));   // 32 pages from `first` on, a lane each; behind the last key: the last one
        auto fetch_q = [&](int g) {
          if ((p.pair ? p.cnt(g) : 1 - g) == 0) return true;
          if (!gemm_wait_warp(smem_u32(&q_empty[g]), (cq[g] & 1) ^ 1, abortp)) return false;
          ++cq[g];
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[g], T::CH * a.G * a.tile_tokens * 128);
            for (int c = 0; c < T::CH; ++c)
              gemm_tma_3d<1>(smQ + g * T::TILE + c * 16384, &map_q, smem_u32(&q_full[g]), c * 64, p.head * a.G, p.row0 + g * a.tile_tokens);
          }
          return true;
        };
        auto fetch = [&](const CUtensorMap* map, uint32_t dst, uint64_t* full, int page0, int page1) {
          if (lane) return;
          mbar_arrive_expect_tx(full, T::TILE);
          for (int r = 0; r < 2; ++r)   // a page at a time
            for (int c = 0; c < T::CH; ++c) fap_tma_4d(dst + c * 16384 + r * 8192, map, smem_u32(full), c * 64, 0, p.head, r ? page1 : page0);
        };
        // In the order in which the MMAs ask for them.
        if (!(alive = fetch_q(0))) break;
        for (int j = 0; j < p.n; ++j, ++ck) {
          const int i = ck & 1, ph = (ck >> 1) & 1;
          if (2 * (p.k0 + j) >= first + 32) {
            first += 32;
            ids = __ldg(pages + min(first + lane, last_page));
          }
          const int page0 = __shfl_sync(0xffffffffu, ids, 2 * (p.k0 + j) - first), page1 = __shfl_sync(0xffffffffu, ids, 2 * (p.k0 + j) + 1 - first);
          if (!(alive = gemm_wait_warp(smem_u32(&k_empty[i]), ph ^ 1, abortp))) break;
          fetch(&map_k, smK + i * T::TILE, &k_full[i], page0, page1);
          if (j == 0 && !(alive = fetch_q(1))) break;
          if (!(alive = gemm_wait_warp(smem_u32(&v_empty[i]), ph ^ 1, abortp))) break;
          fetch(&map_v, smV + i * T::TILE, &v_full[i], page0, page1);
        }
      }
    }
    // ------------------------------------------------------------------------------------------------ MMAs
    if (warp == 9) {
      // the whole warp walks the loop, one elected lane issues (as in the prompt's kernel)
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t dq0 = umma_desc_sw128(smQ), dk0 = umma_desc_sw128(smK), dv0 = fap_desc_mn(smV);
      bool alive = true;   // a lane's own: once a wait expires it only keeps the lane from issuing
      int c[2] = {0, 0}, cq[2] = {0, 0}, ck = 0;   // tiles of group g, pieces with a query tile g, tiles of K and V, before this piece
      auto qk = [&](int g, int tile, int slot) {   // S_g = Q_tile K^T
        const uint64_t dq = dq0 + (uint64_t)(tile * (T::TILE >> 4)), dk = dk0 + (uint64_t)(slot * (T::TILE >> 4));
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          umma_bf16(tm + COL_S + g * 128, dq + (k >> 2) * 1024 + 2 * (k & 3), dk + (k >> 2) * 1024 + 2 * (k & 3), ID_S, k > 0 ? 1u : 0u);
        fap_commit(&s_full[g]);
      };
      auto pv = [&](int g, int slot, bool first) {
        const uint64_t dv = dv0 + (uint64_t)(slot * (T::TILE >> 4));
#pragma unroll
        for (int k = 0; k < 8; ++k)   // 16 keys: 8 columns of P, two 8-key atoms of V
          umma_f16_ts(tm + COL_O + g * D, tm + COL_S + g * 128 + 8 * k, dv + k * (2048 >> 4), ID_O, (!first || k > 0) ? 1u : 0u);
        fap_commit(&o_full[g]);
      };
      auto wait_k = [&](int t) { alive &= gemm_wait(smem_u32(&k_full[t & 1]), (t >> 1) & 1, abortp); };
      auto wait_v = [&](int t) { alive &= gemm_wait(smem_u32(&v_full[t & 1]), (t >> 1) & 1, abortp); };
      // the first scores of group g of piece p, whose key tiles begin at tile t and whose query tiles are number q0, q1
      auto open = [&](const ChunkPiece& p, int g, int t, int q0, int q1) {
        const int tile = p.pair ? g : 0, step = p.pair ? 0 : g;
        alive &= gemm_wait(smem_u32(&q_full[tile]), (tile ? q1 : q0) & 1, abortp);
        wait_k(t + step);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_one() && alive) {
          qk(g, tile, (t + step) & 1);
          if (!p.pair) fap_commit(&k_empty[(t + step) & 1]);                  // (of a pair, both tiles read the same keys)
          if (p.pair ? p.cnt(g) == 1 : step == p.n - 1) fap_commit(&q_empty[tile]);   // behind the last scores Q's place is free
        }
      };
      bool ahead[2] = {false, false};              // this piece's first scores of group g are issued already
      int at = begin;
      ChunkPiece p, next;
      bool more = chunk_piece(a, at, end, next);
      while (more) {
        p = next;
        more = chunk_piece(a, at, end, next);
        const int tn = ck + p.n;                   // the next piece's first key tile
        const int nq0 = cq[0] + (p.pair ? p.cnt0 > 0 : 1), nq1 = cq[1] + (p.pair && p.cnt1 > 0);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (p.cnt(g) > 0 && !ahead[g]) open(p, g, ck, cq[0], cq[1]);
          ahead[g] = false;
        }
        // the next piece's scores, while this one's last tiles and its O are worked on
        auto go_on = [&](int g) {
          if (more && next.cnt(g) > 0) {
            open(next, g, tn, nq0, nq1);
            ahead[g] = true;
          }
        };
        if (p.pair) {
          if (elect_one() && alive) fap_commit(&k_empty[ck & 1]);
          for (int j = 0; j < p.n; ++j) {
            const int t = ck + j, i = t & 1, i2 = (t + 1) & 1;
            wait_v(t);
            if (j + 1 < p.n) wait_k(t + 1);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int ng = p.cnt(g);
              if (j < ng) {
                alive &= gemm_wait(smem_u32(&p_full[g]), (c[g] + j) & 1, abortp);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one() && alive) {
                  pv(g, i, j == 0);
                  if (j + 1 < ng) {
                    qk(g, g, i2);
                    if (j + 2 == ng) fap_commit(&q_empty[g]);
                  }
                }
                if (j + 1 == ng) go_on(g);
              }
            }
            if (elect_one() && alive) {
              fap_commit(&v_empty[i]);
              if (j + 1 < p.n) fap_commit(&k_empty[i2]);
            }
          }
        } else {
          for (int j = 0; j < p.n; ++j) {
            const int t = ck + j, g = j & 1;
            wait_v(t);
            alive &= gemm_wait(smem_u32(&p_full[g]), (c[g] + (j >> 1)) & 1, abortp);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one() && alive) {
              pv(g, t & 1, j < 2);
              fap_commit(&v_empty[t & 1]);
            }
            if (j + 2 < p.n) {
              wait_k(t + 2);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              if (elect_one() && alive) {
                qk(g, 0, t & 1);
                fap_commit(&k_empty[t & 1]);
                if (j + 3 == p.n) fap_commit(&q_empty[0]);
              }
            } else {
              go_on(g);
            }
          }
        }
        c[0] += p.cnt0; c[1] += p.cnt1; ck = tn;
        cq[0] = nq0; cq[1] = nq1;
      }
    }
    // ------------------------------------------------------------------------------------------------ rows behind the last request's
    if (warp == 10 && a.rest) {
      const int row_words = a.Hq * D / 8;   // of 16 bytes
      for (long long e = ((long long)__ldg(a.row_starts + a.requests) + blockIdx.x) * row_words; e < (long long)a.rows * row_words; e += (long long)gridDim.x * row_words)
        for (int i = lane; i < row_words; i += 32) reinterpret_cast<uint4*>(a.out)[e + i] = make_uint4(0, 0, 0, 0);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (*abortp) gemm_drain();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
}

template <int D>
static cudaError_t launch_chunk(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const ChunkArgs& a, cudaStream_t st) {
  using T = FapTile<D>;
  static std::atomic<unsigned long long> served{0};
  const cudaError_t set = once_per_device(served, [] {
    cudaFuncAttributes at;
    const cudaError_t e = cudaFuncGetAttributes(&at, chunk_attn_kernel<D>);
    if (e != cudaSuccess) return e;
    // the warps' register shares must fit what the block is launched with, or they would wait for registers for good
    if (at.numRegs * T::THREADS < 8 * 32 * 216 + 4 * 32 * 64) return cudaErrorInvalidConfiguration;
    return cudaFuncSetAttribute(chunk_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
  });
  if (set != cudaSuccess) return set;
  count_launch();
  return launch_pdl(chunk_attn_kernel<D>, dim3((unsigned)(num_sms() < kStepMaxCtas ? num_sms() : kStepMaxCtas)), dim3(T::THREADS), T::SMEM, st, mq, mk, mv, a);
}

}  // namespace pie

extern "C" {

using namespace pie;

size_t pie_chunk_attn_workspace_bytes(const pie_step_dims* d, int D) {
  if (step_dims_status(d) || (D != 64 && D != 128)) return 0;
  return kStepMaxCtas * 4 + (size_t)2 * kStepMaxCtas * (D == 128 ? kChunkRecord<128> : kChunkRecord<64>) * 4;
}

int pie_chunk_attn(void* out, const pie_head_rows* q, const void* kpool, const void* vpool, const pie_kv_layout* kv, const int32_t* plan, const pie_step_dims* d, int D,
                   float scale, int rest, void* workspace, size_t workspace_bytes, void* stream) {
  if (int s = step_dims_status(d)) return s;
  if (!out || !q || !q->p || !kpool || !vpool || !kv || !plan) return PIE_ENULL;
  if ((D != 64 && D != 128) || !(scale > 0.f) || scale > 3.4028234e38f / 1.5f || kv->tok_stride <= 0 || kv->tok_stride % 8 || kv->head_stride % 8 || q->stride_h % 8 ||
      q->stride_l % 8 || (d->rows > 1 && q->stride_l <= 0) || (d->Hq > 1 && q->stride_h <= 0) || (d->Hkv > 1 && kv->head_stride <= 0))
    return PIE_EINVAL_SHAPE;
  for (const void* p : {(const void*)out, q->p, kpool, vpool, (const void*)plan, (const void*)workspace})
    if (reinterpret_cast<uintptr_t>(p) & 15) return PIE_EALIGN;
  if (!workspace || workspace_bytes < pie_chunk_attn_workspace_bytes(d, D)) return PIE_EWORKSPACE;
  const StepLayout l = step_layout(*d);
  ChunkArgs a;
  a.out = (uint16_t*)out; a.Hq = d->Hq; a.G = d->Hq / d->Hkv; a.tile_tokens = l.tile_tokens; a.rows = d->rows; a.requests = d->requests;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.ranges = plan + l.ranges; a.table = plan + l.block_table; a.row_starts = plan + l.row_starts;
  a.pieces = reinterpret_cast<const StepPiece*>(plan + l.pieces);
  a.blocks = d->blocks; a.rest = rest;
  a.count = (unsigned int*)workspace;
  a.part = (float*)((uint8_t*)workspace + kStepMaxCtas * 4);
  const GemmEncodeFn fn = gemm_encode_fn();
  if (!fn) return PIE_ECUDA;
  CUtensorMap maps[3];
  const cuuint32_t one[4] = {1, 1, 1, 1};
  {   // a query tile: 64 features of G heads of tile_tokens rows
    const long long head = (d->Hq > 1 ? q->stride_h : D) * 2, row = (d->rows > 1 ? q->stride_l : (long long)d->Hq * D) * 2;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)d->Hq, (cuuint64_t)d->rows}, strides[2] = {(cuuint64_t)head, (cuuint64_t)row};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)a.tile_tokens};
    if (fn(&maps[0], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q->p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return PIE_EUNSUPPORTED;
  }
  for (int i = 0; i < 2; ++i) {   // a page of one head: 64 features of its 64 slots
    const long long tok = kv->tok_stride * 2, head = d->Hkv > 1 ? kv->head_stride * 2 : tok;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)kStepPage, (cuuint64_t)d->Hkv, (cuuint64_t)d->pages};
    const cuuint64_t strides[3] = {(cuuint64_t)tok, (cuuint64_t)head, (cuuint64_t)(kStepPage * tok)};
    const cuuint32_t box[4] = {64, 64, 1, 1};
    if (fn(&maps[1 + i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(i ? vpool : kpool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return PIE_EUNSUPPORTED;
  }
  return status_of(D == 128 ? launch_chunk<128>(maps[0], maps[1], maps[2], a, (cudaStream_t)stream) : launch_chunk<64>(maps[0], maps[1], maps[2], a, (cudaStream_t)stream));
}

}  // extern "C"
