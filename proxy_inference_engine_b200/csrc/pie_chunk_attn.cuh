// Causal attention of every request's new tokens over its pages (include/pie_b200.h), on the 5th-generation tensor cores.  Compiled with pie_fa_prefill.cu, whose
// tile this is (two softmax groups of four warps, a TMA warp, a warp that issues the MMAs) and whose pipeline word it shares.
//
// Replaces, for the rows of a ragged step, mx.fast.scaled_dot_product_attention with the causal mask of create_attention_mask (PIE/models/base.py:18-53, 92-113).
//
// The rows of a query tile are the query heads of one key / value head, token by token (32 tokens of 4 heads): keys and values are read once for all of them, and a tile
// of few tokens crosses the diagonal in few key tiles.  An item (pie_step_plan.h) is of one of three kinds:
//   * pair: rows in both query tiles.  They walk the same key tiles, one tile's softmax under the other's MMAs, as in the prompt's kernel -- bound by softmax and tensor pipe.
//   * one tile of more rows than that has: the groups take every other key tile of it, each with its own maximum, sum and accumulator, which meet at the end through tensor
//     memory (the groups' warps read the same lanes).
//   * few, up to 64 rows, 48 at head size 128 (an answer's token, drafted ones): every other key tile as well, but turned around.  S^T = K Q^T has a key a lane and the rows, padded to 16,
//     for its columns; P goes to shared memory as the B operand of O^T = V^T P^T.  The softmax of 4 rows is then 4 exponentials of each of the 128 threads instead of 128 of four of
//     them, and the MMAs are as narrow as the rows: bound by the stream of keys and values.  (A row a lane: one warp a group does all the work, and both of them on the same
//     quarter of the SM; head size 64 40 x 12000 keys 259 us, 59 % of the stream's rate.)  A column's maximum is taken over all lanes only where some score exceeds the reference by
//     2^8, which the group finds by a vote; the sums over the lanes wait for the end.
// Weights are multiplied with V as bf16, and so rounded, in the two kinds of more rows as in the prompt's kernel (2^-8 of a weight; pairs would take the tensor pipe,
// which bounds there, half as long again).  The few rows' are pairs of bf16, first and second 8 bits, as in the decode kernels: an answer must not depend on which of them it is given.  A row's
// second halves are eight rows of P behind its first ones -- so both lie at offsets known beforehand -- and the same MMA, twice as wide, gives them columns of their own, added up with the results.
// (Two MMAs into the same columns: head size 64, 40 answers with up to five drafts over 12000 keys 236 us, 220 so; rounded once: 191.  Head size 128: 309 and 305.  Shared memory has room
// for 48 rows' pairs at head size 128; 64 / 8 heads, 16 answers with up to seven drafts over 4000 keys, the longest as one tile 79.7 us, all turned around with weights rounded once 75.9.)
// A CTA per SM walks the pieces that the plan dealt out to it.  A piece of a cut item leaves its maxima, sums and unnormalised results (fp32) in its CTA's place of the
// workspace, and the last CTA of the item to arrive adds all pieces up in their order: the same bits whichever that is.
// Keys that a row must not see get weight 0; values behind the item's last key are cleared in shared memory, since 0 * NaN is not 0.
// Every wait is bounded (pie_gemm.cuh); a warp whose wait ran out does nothing more, but walks on through the barriers of the softmax warps.
// Device time in a row of such calls, inputs not in L2, 32 query / 8 kv heads: D 128, 2048 tokens behind 15000 460 us (1170 TFLOP/s, of cuBLAS's 1638 in a burst; the tensor pipe is
// busy for 54 % of it, as in the prompt's kernel one tile's softmax is covered by the other's products in part); 16 answers with up to five drafted tokens over 4000 keys 51.6 (4.4 TB/s),
// 40 over 12000 309 (6.4 TB/s), one with four over 9000 26.3; D 64, three portions of 700 tokens beside 29 answers over 1500 keys 83.9, 40 answers over 12000 220 (4.5 TB/s).  Short
// steps pay 4 us from the launch to the first scores, some 3 at each turn from one piece to the next and 5 at the end: results, one counter, the last CTA's sums.
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
  float* part;                 // [2 CTAs] records
  int rest;
  int few_tokens;              // tokens of an item of the turned kind, at most
  // 8-bit pages: codes [pages, Hkv, 64, D], scales [pages, Hkv]
  const uint8_t *k8, *v8;
  const float *k_scales, *v_scales;
  int Hkv;
};
template <int D>
constexpr int kChunkRecord = 256 * D + 512;   // floats: results, [64 rows][D] of the turned kind, [D / 4][256 rows][4] of the others; [256] maxima and sums
constexpr int kChunkFew = 64;                 // rows of an item of the turned kind, at most (ChunkTile::FEW)
constexpr int kChunkList = 32;                // pieces held in shared memory; a CTA that has more reads them where they are

template <int D, bool F8 = false>
struct ChunkTile {
  static constexpr int CH = D / 64, TILE = 128 * D * 2;          // 64-feature chunks of a row, bytes of 128 rows
  static constexpr int RK = F8 ? (D == 64 ? 2 : 1) : D == 64 ? 4 : 2;   // tiles of K
  static constexpr int RV = F8 ? 2 : RK;                         // tiles of V
  static constexpr int FEW = F8 ? 32 : D == 64 ? 64 : 48;        // rows of an item of the turned kind, at most: as shared memory has room for their weights
  static constexpr int HALVES = (FEW + 31) / 32;                 // of 32 rows
  static constexpr int PCHUNK = 2 * FEW * 128;                   // bytes of 64 keys of a group's P of the turned kind: eight rows' first halves, their second halves, ...
  static constexpr int P = 2 * PCHUNK;
  static constexpr int Q1 = TILE > 2 * P ? TILE : 2 * P;         // the second query tile; the turned kind's P
  static constexpr int PAGE = 64 * D, PAGES = F8 ? (D == 64 ? 16 : 6) : 1;   // bytes of a page of one head in 8 bits, and how many of them wait to be converted
  static constexpr int SMEM = 1024 + TILE + Q1 + (RK + RV) * TILE + (F8 ? PAGES * PAGE : 0);
  static constexpr int THREADS = F8 ? 512 : 384;
  // warps 0-7 softmax, 8 TMA, 9 MMAs, 10 scales (8-bit pages), W_REST rows of nobody, 12-15 conversion (8-bit pages)
  static constexpr int W_REST = F8 ? 11 : 10;
  // Registers, which must not exceed what the block is launched with: 384 x 168 = 64512, 256 x 216 and 128 x 64 are 63488; 512 x 128 = 65536 = 256 x 208 and 256 x 48
  static constexpr int REGS_SOFTMAX = F8 ? 208 : 216, REGS_REST = F8 ? 48 : 64;
};
constexpr int kChunkScales = 4;               // 8-bit pages: key tiles of a group whose scales are held

enum ChunkKind { CHUNK_PAIR, CHUNK_ONE, CHUNK_FEW };
// a piece as the roles walk it
struct ChunkPiece {
  int row0, pos0, tokens, request, head, k0, n, first, pieces, kind;
  int cnt0, cnt1;              // key tiles of either group
  __device__ __forceinline__ int cnt(int g) const { return g ? cnt1 : cnt0; }
};
__device__ __forceinline__ const int4* chunk_words(const ChunkArgs& a, const int4* list, int begin, int at) {
  return at - begin < kChunkList ? list + 3 * (at - begin) : reinterpret_cast<const int4*>(a.pieces + at);
}
// false: an empty one
__device__ __forceinline__ bool chunk_read(const ChunkArgs& a, const int4& x, const int4& y, const int4& z, ChunkPiece& p) {
  p.row0 = x.x; p.pos0 = x.y; p.tokens = x.z; p.request = x.w;
  p.head = y.x; p.k0 = y.y; p.n = y.z - y.y; p.first = y.w;
  p.pieces = z.x;
  p.kind = p.tokens > a.tile_tokens ? CHUNK_PAIR : p.tokens <= a.few_tokens ? CHUNK_FEW : CHUNK_ONE;
  if (p.kind == CHUNK_PAIR) {
    p.cnt0 = max(0, min(p.n, (p.pos0 + a.tile_tokens - 1) / kStepTile + 1 - p.k0));
    p.cnt1 = p.n;
  } else {
    p.cnt0 = (p.n + 1) / 2;
    p.cnt1 = p.n / 2;
  }
  return p.n > 0;
}
__device__ __forceinline__ bool chunk_piece(const ChunkArgs& a, const int4* list, int begin, int& at, int end, ChunkPiece& p) {
  while (at < end) {
    const int4* const e = chunk_words(a, list, begin, at++);
    if (chunk_read(a, e[0], e[1], e[2], p)) return true;
  }
  p.n = p.cnt0 = p.cnt1 = 0;
  return false;
}
__device__ __forceinline__ void chunk_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }   // the eight softmax warps
__device__ __forceinline__ void chunk_group_sync(int g) {
  if (g) asm volatile("bar.sync 3, 128;" ::: "memory");
  else asm volatile("bar.sync 2, 128;" ::: "memory");
}
template <int BAR>
__device__ __forceinline__ uint32_t chunk_any(uint32_t mine) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(any) : "r"(mine), "n"(BAR) : "memory");
  return any;
}
__device__ __forceinline__ bool chunk_group_any(int g, bool mine) { return (g ? chunk_any<3>(mine) : chunk_any<2>(mine)) != 0; }
__device__ __forceinline__ void chunk_st16(uint32_t taddr, const float* v) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(u[0]), "r"(u[1]), "r"(u[2]),
      "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]),
      "r"(taddr) : "memory");
}
__device__ __forceinline__ void chunk_ld16(uint32_t taddr, float* v) { tmem_ld16(taddr, *reinterpret_cast<uint32_t(*)[16]>(v)); }   // not waited for
__device__ __forceinline__ int chunk_order(float x) {   // integers in the order of the numbers
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float chunk_unorder(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
// what the turned kind keeps of its rows
struct ChunkFew {
  int best[2][4][kChunkFew];      // a warp's largest score of each row, in chunk_order
  float m[2][kChunkFew];          // reference point of a group's sums, -inf: none yet
  float less[2][kChunkFew];       // what is added to a scaled score: -m, or 0
  float factor[2][kChunkFew];     // by which the sums and results of a row that moved shrink
  float sum[2][4][kChunkFew];     // a warp's part of a row's sum
  float2 share[kChunkFew];        // factors of the two groups' results
  int row[kChunkFew];             // a row's place among the step's rows x heads
};

// Adds up the pieces of a cut item: by the eight softmax warps of the CTA that came last.
template <int D>
__device__ __forceinline__ void chunk_merge(uint16_t* out, const float* part, int first, int pieces, int tokens, int row0, int head, int Hq, int G, bool few) {
  const int tid = threadIdx.x;
  // the item's pieces: the one that opens it, and the ones of the CTAs behind, in order
  const float* const rec0 = part + (size_t)(2 * first + 1) * kChunkRecord<D>;
  auto piece = [&](int i) { return rec0 + (i == 0 ? 0 : i * 2 * (ptrdiff_t)kChunkRecord<D> - kChunkRecord<D>); };
  const int rows = tokens * G;
  // What this costs is trips to L2 (and instructions that are run once), so all loads of a step are under way together.
  auto store = [&](int q, int c4, const float4& o) {
    const int t = q / G;
    *reinterpret_cast<uint2*>(out + ((size_t)(row0 + t) * Hq + head * G + q - t * G) * D + 4 * c4) =
        make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
  };
  // two parts of a row, (m, l, o) <- with (m2, l2, o2); a part without a key (m2 = -inf) may have left no results
  auto join = [](float& m, float& l, float4& o, const float2& ml2, const float4& o2) {
    if (ml2.x == -INFINITY && m != -INFINITY) return;
    const float to = fmaxf(m, ml2.x), f = m == -INFINITY ? 0.f : exp2f(m - to), f2 = exp2f(ml2.x - to);
    l = l * f + ml2.y * f2;
    o.x = o.x * f + o2.x * f2; o.y = o.y * f + o2.y * f2; o.z = o.z * f + o2.z * f2; o.w = o.w * f + o2.w * f2;
    m = to;
  };
  if (!few) {   // a row a thread, eight times four of its features at a time
    if (tid < rows) {
      const int from = 256 * D + 2 * tid;
#pragma unroll 1
      for (int c0 = 0; c0 < D / 4; c0 += 8) {
        float4 o[8];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int i = 0; i < pieces; ++i) {
          float4 v[8];
          const float2 mi = __ldcg(reinterpret_cast<const float2*>(piece(i) + from));
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = __ldcg(reinterpret_cast<const float4*>(piece(i) + ((size_t)(c0 + k) * 256 + tid) * 4));
          float to = m, sum = l;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            to = m; sum = l;
            join(to, sum, o[k], mi, v[k]);
          }
          m = to; l = sum;
        }
        const float inv = 1.f / l;
#pragma unroll
        for (int k = 0; k < 8; ++k) store(tid, c0 + k, make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv));
      }
    }
  } else {                     // four features of a row a lane, eight pieces at a time
    constexpr int LANES = D / 4, STEP = 256 / LANES;
#pragma unroll 1
    for (int q = tid / LANES; q < rows; q += STEP) {
      const int c4 = tid % LANES;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int i0 = 0; i0 < pieces; i0 += 8) {
        float4 v[8];
        float2 mi[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float* const at_piece = piece(min(i0 + k, pieces - 1));
          mi[k] = __ldcg(reinterpret_cast<const float2*>(at_piece + 256 * D + 2 * q));
          v[k] = __ldcg(reinterpret_cast<const float4*>(at_piece + q * D + 4 * c4));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i0 + k < pieces) join(m, l, o, mi[k], v[k]);
      }
      const float inv = 1.f / l;
      store(q, c4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
  }
}

// 16 codes of 8 bits as bf16, exactly: the code's bits in the places of a bf16's are a number 2^120 times smaller (and e4m3's subnormals bf16's)
__device__ __forceinline__ uint32_t chunk_widen(uint32_t w, uint32_t sel) {
  const uint32_t x = __byte_perm(w, 0, sel), y = ((x >> 4) & 0x07f007f0u) | (x & 0x80008000u);
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(y), "r"(0x7b807b80u));
  return d;
}
__device__ __forceinline__ void chunk_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <int D, bool F8>
__global__ void __launch_bounds__(ChunkTile<D, F8>::THREADS, 1)
chunk_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_few, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ChunkArgs a) {
  using T = ChunkTile<D, F8>;
  constexpr int RK = T::RK, RV = T::RV;
  constexpr uint32_t ID_S = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t ID_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t ID_FEW = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);   // | N
  constexpr int COL_S = 0, COL_O = 256, OST = 128;   // + g * 128, + g * OST
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[RK], k_empty[RK], v_full[RV], v_empty[RV], s_full[2], p_full[2], o_full[2];
  // 8-bit pages: pages as they lie, scales of a group's key tiles, products behind which the turned kind's P is free (pieces of that kind in turn)
  __shared__ __align__(8) uint64_t c_full[T::PAGES], c_empty[T::PAGES], sc_full[2][F8 ? kChunkScales : 1], sc_empty[2][F8 ? kChunkScales : 1], turn_free[2];
  __shared__ __align__(16) float sc[2][F8 ? kChunkScales : 1][8];   // of the two pages: scores to log2 units, log2 of the values' scale, its reciprocal, itself
  __shared__ __align__(16) int4 list[3 * kChunkList];
  __shared__ __align__(16) ChunkFew few;
  __shared__ float2 ml[2][128];           // a row's maximum and sum: of the two groups of a tile, of the rows of a cut item
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, last_flag;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  // (The turned kind's P lies where Q1 does.  Its V^T has 128 rows whatever the head size: at 64 the upper ones are what lies 16 KB behind, so V does not lie last.)
  const uint32_t smV = base, smK = smV + RV * T::TILE, smQ = smK + RK * T::TILE, smQ1 = smQ + T::TILE, smC = smQ1 + T::Q1;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < RK; ++i) { mbar_init(&k_full[i], F8 ? 4 : 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < RV; ++i) { mbar_init(&v_full[i], F8 ? 4 : 1); mbar_init(&v_empty[i], 1); }
    if (F8) {
      for (int i = 0; i < T::PAGES; ++i) { mbar_init(&c_full[i], 1); mbar_init(&c_empty[i], 4); }
      for (int i = 0; i < 2 * kChunkScales; ++i) { mbar_init(&sc_full[0][0] + i, 1); mbar_init(&sc_empty[0][0] + i, 4); }
      for (int i = 0; i < 2; ++i) mbar_init(&turn_free[i], 1);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 8 && lane < (F8 ? 2 : 4)) tma_prefetch_desc(lane == 0 ? &map_q : lane == 1 ? &map_few : lane == 2 ? &map_k : &map_v);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot;
  volatile int* const abortp = &abort_flag;
  pdl_launch_dependents();
  pdl_wait();   // (the set-up above ran under the end of the launch before this one)
  const int begin = __ldg(a.ranges + 2 * blockIdx.x), end = __ldg(a.ranges + 2 * blockIdx.x + 1);
  // The CTA's pieces.  (The TMA warp reads the first one where it is and asks for its keys meanwhile.)
  if (warp != 8) {
    for (int i = warp < 8 ? tid : tid - 32; i < 3 * min(end - begin, kChunkList); i += T::THREADS - 32)
      list[i] = __ldg(reinterpret_cast<const int4*>(a.pieces + begin) + i);
    asm volatile("bar.sync 4, %0;" ::"n"(T::THREADS - 32) : "memory");
    if (end - begin > 1) asm volatile("bar.arrive 5, %0;" ::"n"(T::THREADS) : "memory");
  }

  // All barriers are counted over the CTA's pieces: a role keeps the number of key tiles (of its group, of K and V) before its piece.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(T::REGS_SOFTMAX));
    // ------------------------------------------------------------------------------------------------ softmax of group g
    const int g = warp >> 2, quad = warp & 3, r = quad * 32 + lane, tok = r / a.G;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t tS = tmem + COL_S + g * 128 + lanes, tO = tmem + COL_O + lanes;
    int c[2] = {0, 0}, cv = 0;     // key tiles of either group, tiles of V, before this piece
    bool alive = true;
    int at = begin;
    ChunkPiece p;
    // values behind the item's last key may be anything: this thread's row of the key tile they lie in
    auto clear_tail = [&](int step, int tail) {
      const int v = cv + step;
      alive = alive && gemm_wait_warp(smem_u32(&v_full[v % RV]), (v / RV) & 1, abortp);
      if (alive && r >= tail)
#pragma unroll
        for (int q = 0; q < 8 * T::CH; ++q)
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(smV + (v % RV) * T::TILE + (q >> 3) * 16384 + r * 128 + (q & 7) * 16), "r"(0) : "memory");
      fence_proxy_async();
    };
    // 8-bit pages: the scales of this group's key tile n, before its scores are there (both pages'; (c, log2 v, 1 / v, v) of page h at h, 2 + h, ...)
    auto take_scales = [&](int n, float (&to)[8]) {
      const int i = n % kChunkScales;
      alive = alive && gemm_wait_warp(smem_u32(&sc_full[g][i]), (n / kChunkScales) & 1, abortp);
      *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(sc[g][i]);
      *reinterpret_cast<float4*>(to + 4) = *reinterpret_cast<const float4*>(sc[g][i] + 4);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc_empty[g][i]);
    };
    // Registers are short where a thread holds a row of scores: the loops keep a few numbers, and the piece is read again behind them.
    auto read_again = [&]() {
      const volatile int* const e = reinterpret_cast<const volatile int*>(chunk_words(a, list, begin, at - 1));
      p.row0 = e[0]; p.pos0 = e[1]; p.tokens = e[2]; p.head = e[4]; p.first = e[7]; p.pieces = e[8];
    };
    while (chunk_piece(a, list, begin, at, end, p)) {
      const int keys = p.pos0 + p.tokens, tail = keys & 127, tail_step = tail ? (keys - 1) / 128 - p.k0 : -1, cnt = p.cnt(g);
      if (p.kind == CHUNK_FEW) {
        // ---------------------------------------------------------------------------------- a key a lane, a row a column
        const int rows = p.tokens * a.G;
        const int beyond = p.k0 * 128 + r - p.pos0, edge_step = (p.pos0 + 1) / 128 - p.k0;   // the first key tile with a key that some row must not see
        const uint32_t sp = smQ1 + g * T::P + (r >> 6) * T::PCHUNK + (r & 7) * 2;
        const int chunk16 = (r & 63) >> 3;
        float l[32 * T::HALVES];
#pragma unroll
        for (int n = 0; n < 32 * T::HALVES; ++n) l[n] = 0.f;
        for (int i = 0; i < cnt; ++i) {
          const int step = 2 * i + g;
          float to_log2 = a.scale_log2e, value = 1.f;   // of this lane's key: of its page
          if constexpr (F8) {
            float of[8];
            take_scales(c[g] + i, of);
            to_log2 = quad < 2 ? of[0] : of[1];
            value = quad < 2 ? of[6] : of[7];
          }
          alive = alive && gemm_wait_warp(smem_u32(&s_full[g]), (c[g] + i) & 1, abortp);
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          float s[32];
          // 32 rows' scores; those of rows in front of `cut`, which this lane's key lies beyond, and of rows without a token do not count
          auto load = [&](int half) {
            chunk_ld16(tS + 32 * half, s);
            if (32 * half + 16 < rows) chunk_ld16(tS + 32 * half + 16, s + 16);
            tmem_ld_wait();
            if (step >= edge_step) {
              const int cut = (beyond + step * 128) * a.G - 32 * half;   // (a key that far beyond the first row's own: the place in the cache times G may not fit)
#pragma unroll
              for (int n = 0; n < 32; ++n)
                if (n < cut) s[n] = -INFINITY;
            }
            if (rows & 3)   // (four rows are worked on at a time; what P has for the rows behind those does not matter)
#pragma unroll
              for (int n = 0; n < 32; ++n)
                if (32 * half + n >= rows) s[n] = -INFINITY;
          };
          // the weights in the scores' place, and the largest
          auto weigh = [&](int half) {
            float mx = 0.f;
#pragma unroll
            for (int n = 0; n < 32; n += 4) {
              if (32 * half + n >= rows) break;
              const float4 less = *reinterpret_cast<const float4*>(&few.less[g][32 * half + n]);
              s[n] = fap_exp2(fmaf(s[n], to_log2, less.x));
              s[n + 1] = fap_exp2(fmaf(s[n + 1], to_log2, less.y));
              s[n + 2] = fap_exp2(fmaf(s[n + 2], to_log2, less.z));
              s[n + 3] = fap_exp2(fmaf(s[n + 3], to_log2, less.w));
              mx = fmaxf(fmaxf(mx, fmaxf(s[n], s[n + 1])), fmaxf(s[n + 2], s[n + 3]));
            }
            return mx;
          };
          // four rows' weights into the swizzled tile: 128 bytes a row, its 16-byte chunks in another order
          auto put = [&](int row, uint32_t w01, uint32_t w23) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t w = k < 2 ? w01 : w23;
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(sp + (row + k) * 128 + ((chunk16 ^ ((row + k) & 7)) << 4)), "h"((uint16_t)(k & 1 ? w >> 16 : w)) : "memory");
            }
          };
          bool over = i == 0;
          if (T::HALVES > 1 && i > 0 && rows > 32) {
            load(1);
            over = weigh(1) > 256.f;
          }
          load(0);
          if (i > 0) over = weigh(0) > 256.f || over;
          // the reference of a row moves where a score exceeds it by 8 (log2 units: a weight of 256): same sums, and mostly the lanes need not know of one another
          if (chunk_group_any(g, over)) {
#pragma unroll
            for (int half = 0; half < T::HALVES; ++half)
              if (32 * half < rows) {
                if (half || i > 0) load(half);
                int mine = 0;
#pragma unroll
                for (int n = 0; n < 32; ++n) {
                  if (32 * half + n >= rows) break;
                  const int v = __reduce_max_sync(0xffffffffu, chunk_order(F8 ? s[n] * to_log2 : s[n]));
                  if (lane == n) mine = v;
                }
                few.best[g][quad][32 * half + lane] = mine;
              }
            chunk_group_sync(g);
            if (quad == 0)
              for (int n = lane; n < rows; n += 32) {
                const float was = i == 0 ? -INFINITY : few.m[g][n];
                const float now = chunk_unorder(max(max(few.best[g][0][n], few.best[g][1][n]), max(few.best[g][2][n], few.best[g][3][n]))) * (F8 ? 1.f : a.scale_log2e);
                const bool move = i == 0 || now > was + 8.f;
                const float m = move ? now : was;
                few.factor[g][n] = !move ? 1.f : was == -INFINITY ? 0.f : fap_exp2(was - m);
                few.m[g][n] = m;
                few.less[g][n] = m == -INFINITY ? 0.f : -m;
              }
            chunk_group_sync(g);
            if (i > 0) {
              // O holds the tiles before this one once their product has finished
              alive = alive && gemm_wait_warp(smem_u32(&o_full[g]), (c[g] + i - 1) & 1, abortp);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
              for (int b = 0; b < T::FEW / 8; ++b)
                if (8 * b < rows) {
                  float o[16];
                  chunk_ld16(tO + g * OST + 16 * b, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int n = 0; n < 8; ++n) {
                    const float f = few.factor[g][8 * b + n];
                    l[8 * b + n] *= f;
                    o[n] *= f;
                    o[8 + n] *= f;
                  }
                  chunk_st16(tO + g * OST + 16 * b, o);
                }
              tmem_st_wait();
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            }
            if ((T::HALVES > 1 && rows > 32) || i > 0) load(0);
            weigh(0);
          }
#pragma unroll
          for (int half = 0; half < T::HALVES; ++half)
            if (32 * half < rows) {
              if (half) {
                load(1);
                weigh(1);
              }
#pragma unroll
              for (int n = 0; n < 32; n += 4) {
                if (32 * half + n >= T::FEW || 32 * half + n >= rows) break;
                l[32 * half + n] += s[n]; l[32 * half + n + 1] += s[n + 1]; l[32 * half + n + 2] += s[n + 2]; l[32 * half + n + 3] += s[n + 3];
                if constexpr (F8) { s[n] *= value; s[n + 1] *= value; s[n + 2] *= value; s[n + 3] *= value; }
                const uint32_t w01 = pack_bf16(s[n], s[n + 1]), w23 = pack_bf16(s[n + 2], s[n + 3]);
                const int row = 2 * (32 * half + n) - n % 8;
                put(row, w01, w23);
                put(row + 8, pack_bf16(s[n] - bf16lo(w01), s[n + 1] - bf16hi(w01)), pack_bf16(s[n + 2] - bf16lo(w23), s[n + 3] - bf16hi(w23)));
              }
            }
          if (!F8 && step == tail_step) clear_tail(step, tail);   // (8-bit codes are finite as they are converted)
          fence_proxy_async();
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
        }
        // a row's sum over the warp's lanes: half of the columns a step, until a lane has one
#pragma unroll
        for (int half = 0; half < T::HALVES; ++half)
          if (32 * half < rows) {
            float* const v = l + 32 * half;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
              for (int k = 0; k < o; ++k) {
                const float give = lane & o ? v[k] : v[k + o], keep = lane & o ? v[k + o] : v[k];
                v[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
              }
            few.sum[g][quad][32 * half + lane] = v[0];
          }
        read_again();
        const bool whole = p.pieces == 1;
        float* const rec = a.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == p.first)) * kChunkRecord<D>;
        c[0] += p.cnt0; c[1] += p.cnt1; cv += p.n;
        alive = alive && gemm_wait_warp(smem_u32(&o_full[0]), (c[0] - 1) & 1, abortp);
        if (p.cnt1 > 0) alive = alive && gemm_wait_warp(smem_u32(&o_full[1]), (c[1] - 1) & 1, abortp);
        chunk_sync();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (tid < rows) {   // (at most 64)
          const float m0 = few.m[0][tid], m1 = p.cnt1 > 0 ? few.m[1][tid] : -INFINITY, m = fmaxf(m0, m1);
          const float f0 = m0 == -INFINITY ? 0.f : fap_exp2(m0 - m), f1 = m1 == -INFINITY ? 0.f : fap_exp2(m1 - m);
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            l0 += few.sum[0][w][tid];
            if (p.cnt1 > 0) l1 += few.sum[1][w][tid];
          }
          const float sum = l0 * f0 + (p.cnt1 > 0 ? l1 * f1 : 0.f), inv = whole ? 1.f / sum : 1.f;
          few.share[tid] = make_float2(f0 * inv, f1 * inv);
          const int t = tid / a.G;
          few.row[tid] = (p.row0 + t) * a.Hq + p.head * a.G + tid - t * a.G;
          if (!whole) __stcg(reinterpret_cast<float2*>(rec + 256 * D + 2 * tid), make_float2(m, sum));
        }
        chunk_sync();
        if (alive && (D == 128 || quad < 2)) {   // (head size 64: nothing in the upper lanes)
#pragma unroll 1
          for (int b = 0; 16 * b < rows; ++b) {
            const int n0 = 16 * b + 8 * g;
            float v[8];
#pragma unroll
            for (int n = 0; n < 8; ++n) v[n] = 0.f;
#pragma unroll 1
            for (int h = 0; h < (p.cnt1 > 0 ? 2 : 1); ++h) {   // the groups' results: by the first halves of the weights, by the second
              float o[16];
              chunk_ld16(tO + h * OST + 2 * n0, o);
              tmem_ld_wait();
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                const float2 f = few.share[n0 + n];
                v[n] += (o[n] + o[8 + n]) * (h ? f.y : f.x);
              }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
              if (n0 + n < rows) {
                if (whole) a.out[(size_t)few.row[n0 + n] * D + r] = f2bf(v[n]);
                else __stcg(rec + (n0 + n) * D + r, v[n]);
              }
          }
        }
      } else {
        // ---------------------------------------------------------------------------------- a row a lane
        const bool pair = p.kind == CHUNK_PAIR;
        const int t0 = pair ? g * a.tile_tokens : 0;                      // the tile's first token of the item
        const bool busy = __any_sync(0xffffffffu, tok < a.tile_tokens && t0 + tok < p.tokens);
        // last key of the piece that this row, the warp's first row sees
        const int lim = p.pos0 + t0 + tok - p.k0 * 128, first_lim = __shfl_sync(0xffffffffu, lim, 0);
        float m = -INFINITY, l = 0.f;
        for (int i = 0; i < cnt; ++i) {
          const int step = pair ? i : 2 * i + g;
          float of[F8 ? 8 : 1];
          if constexpr (F8) take_scales(c[g] + i, of);
          alive = alive && gemm_wait_warp(smem_u32(&s_full[g]), (c[g] + i) & 1, abortp);
          if (!alive) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (busy) {
            float s[128];
#pragma unroll
            for (int q = 0; q < 4; ++q) fap_tmem_ld(tS + 32 * q, s + 32 * q);
            tmem_ld_wait();
            if (step * 128 + 127 > first_lim) {   // a key of this tile lies beyond some row of the warp
              const int last = lim - step * 128;
#pragma unroll
              for (int k = 0; k < 128; ++k)
                if (k > last) s[k] = -INFINITY;
            }
            float mx;
            if constexpr (F8) {   // a page's half of the row at a time
              float x[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int k0 = 64 * (q >> 1) + 32 * (q & 1);
                x[q] = s[k0];
#pragma unroll
                for (int k = 1; k < 32; ++k) x[q] = fmaxf(x[q], s[k0 + k]);
              }
              mx = fmaxf(fmaxf(x[0], x[1]) * of[0], fmaxf(x[2], x[3]) * of[1]);
            } else {
              float x0 = s[0], x1 = s[1], x2 = s[2], x3 = s[3];
#pragma unroll
              for (int k = 4; k < 128; k += 4) {
                x0 = fmaxf(x0, s[k]); x1 = fmaxf(x1, s[k + 1]); x2 = fmaxf(x2, s[k + 2]); x3 = fmaxf(x3, s[k + 3]);
              }
              mx = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * a.scale_log2e;   // (the scale is positive)
            }
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
                fap_tmem_ld(tO + g * OST + c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= f;
                tmem_st32(tO + g * OST + c0, reinterpret_cast<uint32_t*>(o));
              }
              tmem_st_wait();
            }
            const float ms = m == -INFINITY ? 0.f : m;
            f32x2 sc2 = f2_pack(a.scale_log2e, a.scale_log2e), ms2 = f2_pack(-ms, -ms);
            f32x2 l01 = f2_pack(0.f, 0.f), l23 = l01;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              // (8-bit pages: weights times the values' scale, which the row's sum is rid of again)
              if constexpr (F8) {
                sc2 = f2_pack(of[hf], of[hf]);
                ms2 = f2_pack(of[2 + hf] - ms, of[2 + hf] - ms);
                l01 = f2_pack(0.f, 0.f);
                l23 = l01;
              }
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
              if constexpr (F8) {
                float l0, l1;
                f2_unpack(f2_add(l01, l23), l0, l1);
                l += (l0 + l1) * of[4 + hf];
              }
            }
            if constexpr (!F8) {
              float l0, l1;
              f2_unpack(f2_add(l01, l23), l0, l1);
              l += l0 + l1;
            }
            tmem_st_wait();
          }
          if (!F8 && step == tail_step) clear_tail(step, tail);
          if (!alive) break;
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
        }
        read_again();
        const bool whole = p.pieces == 1, live = tok < a.tile_tokens && (p.kind == CHUNK_PAIR ? g * a.tile_tokens : 0) + tok < p.tokens;
        float* const rec = a.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == p.first)) * kChunkRecord<D>;
        c[0] += p.cnt0; c[1] += p.cnt1; cv += p.n;

        // results.  O is read before this warp says that the next piece's first P is there, which its first product, overwriting O, waits for.
        float f0 = 1.f, f1 = 0.f;   // factors of the two accumulators of one tile
        if (pair) {
          if (cnt > 0) alive = alive && gemm_wait_warp(smem_u32(&o_full[g]), (c[g] - 1) & 1, abortp);
        } else {
          ml[g][r] = make_float2(m, l);
          alive = alive && gemm_wait_warp(smem_u32(&o_full[0]), (c[0] - 1) & 1, abortp);
          if (p.cnt1 > 0) alive = alive && gemm_wait_warp(smem_u32(&o_full[1]), (c[1] - 1) & 1, abortp);
          chunk_sync();
          const float2 u = ml[g ^ 1][r];
          const float mx = fmaxf(m, u.x), fm = m == -INFINITY ? 0.f : fap_exp2(m - mx), fu = u.x == -INFINITY ? 0.f : fap_exp2(u.x - mx);
          l = (l == 0.f ? 0.f : l * fm) + (u.y == 0.f ? 0.f : u.y * fu);
          m = mx;
          f0 = g ? fu : fm;
          f1 = g ? fm : fu;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // columns of this group: its own accumulator, or half of both of one tile's
        const int col0 = pair ? 0 : g * (D / 2), col1 = pair ? D : col0 + D / 2, rr = t0 * a.G + r;   // row of the item
        const uint32_t from = pair ? tO + g * OST : tO;
        const bool two = !pair && p.cnt1 > 0;
        if (alive && busy && (cnt > 0 || !pair)) {
          const float inv = whole ? 1.f / l : 1.f;
          uint16_t* const o_row = a.out + ((size_t)(p.row0 + t0 + tok) * a.Hq + p.head * a.G + r - tok * a.G) * D;
#pragma unroll 1
          for (int c0 = col0; c0 < col1; c0 += 32) {
            float o[32];
            fap_tmem_ld(from + c0, o);
            tmem_ld_wait();
            if (two) {
              float u[32];
              fap_tmem_ld(from + OST + c0, u);
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
        if (!whole && live && (pair || g == 0)) __stcg(reinterpret_cast<float2*>(rec + 256 * D + 2 * rr), make_float2(m, l));
      }

      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      if (p.pieces > 1) {
        chunk_sync();
        if (tid == 0) {
          unsigned int before;   // (release and acquire reach, through the barriers, what every warp stored and will read)
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.count + p.first) : "memory");
          last_flag = before == (unsigned)p.pieces - 1;
          if (last_flag) a.count[p.first] = 0;   // for the next launch: nobody else comes
        }
        chunk_sync();
        if (last_flag) chunk_merge<D>(a.out, a.part, p.first, p.pieces, p.tokens, p.row0, p.head, a.Hq, a.G, p.kind == CHUNK_FEW);
      } else if (p.kind != CHUNK_PAIR) {
        chunk_sync();     // both groups have read both accumulators
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(T::REGS_REST));
    // ------------------------------------------------------------------------------------------------ TMA
    if (warp == 8) {
      bool alive = true;
      int cq[2] = {0, 0}, ck = 0;   // pieces with a query tile g, key tiles, before this piece
      int turned = -RV - 1;         // the last key tile of the last piece of the turned kind
      int cp = 0, few_pieces = 0;   // 8-bit pages: pages of K and V, pieces of the turned kind, before this piece
      bool was_few = false;         // the piece before this one was of that kind
      for (int at = begin; alive && at < end; ++at) {
        if (at == begin + 1) asm volatile("bar.sync 5, %0;" ::"n"(T::THREADS) : "memory");   // (the list is there)
        const int4* const e = at == begin ? reinterpret_cast<const int4*>(a.pieces + at) : chunk_words(a, list, begin, at);
        const int4 z = e[2];
        const int lead0 = z.y, lead1 = z.z;   // the pages of its first key tile
        ChunkPiece p;
        if (!chunk_read(a, e[0], e[1], z, p)) continue;
        const int32_t* const pages = a.table + (size_t)p.request * a.blocks;
        const int last_page = (p.pos0 + p.tokens - 1) / kStepPage;
        int first = 2 * p.k0, ids = __ldg(pages + min(first + lane, last_page));   // 32 pages from `first` on, a lane each; behind the last key: the last one
        auto fetch_q = [&](int g) {
          if ((p.kind == CHUNK_PAIR ? p.cnt(g) : 1 - g) == 0) return true;
          if (!gemm_wait_warp(smem_u32(&q_empty[g]), (cq[g] & 1) ^ 1, abortp)) return false;
          ++cq[g];
          // Q1 lies where P of the turned kind did: behind its last product, which frees the last tile of V (where that place was used since, it has)
          if constexpr (F8) {
            // (of pieces before the one before this, the last products are done: their successor's queries have been asked for)
            if (g && was_few && !gemm_wait_warp(smem_u32(&turn_free[(few_pieces - 1) & 1]), ((few_pieces - 1) >> 1) & 1, abortp)) return false;
          } else {
            if (g && ck - turned <= RV && !gemm_wait_warp(smem_u32(&v_empty[turned % RV]), (turned / RV) & 1, abortp)) return false;
          }
          if (lane == 0) {
            const bool few = p.kind == CHUNK_FEW;
            mbar_arrive_expect_tx(&q_full[g], T::CH * a.G * (few ? a.few_tokens : a.tile_tokens) * 128);
            for (int c = 0; c < T::CH; ++c)
              gemm_tma_3d<1>((g ? smQ1 : smQ) + c * 16384, few ? &map_few : &map_q, smem_u32(&q_full[g]), c * 64, p.head * a.G, p.row0 + g * a.tile_tokens);
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
        const int t0 = ck;
        // two pages as they lie, one behind the other in memory each
        auto fetch_codes = [&](const uint8_t* pool, int page0, int page1) {
#pragma unroll
          for (int r = 0; r < 2; ++r, ++cp) {
            const int i = cp % T::PAGES;
            if (!gemm_wait_warp(smem_u32(&c_empty[i]), ((cp / T::PAGES) & 1) ^ 1, abortp)) return false;
            if (lane == 0) {
              mbar_arrive_expect_tx(&c_full[i], T::PAGE);
              chunk_bulk(smC + i * T::PAGE, pool + ((size_t)(r ? page1 : page0) * a.Hkv + p.head) * T::PAGE, T::PAGE, smem_u32(&c_full[i]));
            }
          }
          return true;
        };
        for (int j = 0; j < p.n; ++j, ++ck) {
          if (2 * (p.k0 + j) >= first + 32) {
            first += 32;
            ids = __ldg(pages + min(first + lane, last_page));
          }
          const int page0 = j == 0 ? lead0 : __shfl_sync(0xffffffffu, ids, 2 * (p.k0 + j) - first);
          const int page1 = j == 0 ? lead1 : __shfl_sync(0xffffffffu, ids, 2 * (p.k0 + j) + 1 - first);
          if constexpr (F8) {
            if (!(alive = fetch_codes(a.k8, page0, page1))) break;
            if (j == 0 && !(alive = fetch_q(1))) break;
            if (!(alive = fetch_codes(a.v8, page0, page1))) break;
          } else {
            const int i = ck % RK, iv = ck % RV;
            if (!(alive = gemm_wait_warp(smem_u32(&k_empty[i]), ((ck / RK) & 1) ^ 1, abortp))) break;
            fetch(&map_k, smK + i * T::TILE, &k_full[i], page0, page1);
            if (j == 0 && !(alive = fetch_q(1))) break;
            if (!(alive = gemm_wait_warp(smem_u32(&v_empty[iv]), ((ck / RV) & 1) ^ 1, abortp))) break;
            fetch(&map_v, smV + iv * T::TILE, &v_full[iv], page0, page1);
          }
        }
        if (p.kind == CHUNK_FEW) { turned = t0 + p.n - 1; ++few_pieces; }
        was_few = p.kind == CHUNK_FEW;
      }
    }
    // ------------------------------------------------------------------------------------------------ MMAs
    if (warp == 9) {
      // the whole warp walks the loop, one elected lane issues (as in the prompt's kernel)
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      // descriptors: their upper words are all the same
      constexpr uint64_t UPPER = ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
      const uint32_t dq0 = (uint32_t)umma_desc_sw128(smQ), dq1 = (uint32_t)umma_desc_sw128(smQ1), dk0 = (uint32_t)umma_desc_sw128(smK), dv0 = (uint32_t)fap_desc_mn(smV);
      bool alive = true;   // a lane's own: once a wait expires it only keeps the lane from issuing
      int c[2] = {0, 0}, cq[2] = {0, 0}, ck = 0;   // tiles of group g, pieces with a query tile g, tiles of K and V, before this piece
      int few_pieces = 0;                          // 8-bit pages: pieces of the turned kind before this one
      // scores of group g by query tile `tile`: S_g = Q K^T, or of the turned kind, whose rows' word of the instruction is `wide`, K Q^T
      auto qk = [&](int g, int tile, int t, uint32_t wide) {
        uint32_t dq = tile ? dq1 : dq0, dk = dk0 + (t % RK) * (T::TILE >> 4);
        asm volatile("" : "+r"(dq), "+r"(dk));   // (what is made of them is made here, and not kept in registers that the warp does not have)
        if (wide) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16(tm + COL_S + g * 128, UPPER | (dk + (k >> 2) * 1024 + 2 * (k & 3)), UPPER | (dq + (k >> 2) * 1024 + 2 * (k & 3)), ID_FEW | wide, k > 0 ? 1u : 0u);
        } else {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16(tm + COL_S + g * 128, UPPER | (dq + (k >> 2) * 1024 + 2 * (k & 3)), UPPER | (dk + (k >> 2) * 1024 + 2 * (k & 3)), ID_S, k > 0 ? 1u : 0u);
        }
        fap_commit(&s_full[g]);
      };
      auto pv = [&](int g, int t, bool first, uint32_t wide) {
        uint32_t dv = dv0 + (t % RV) * (T::TILE >> 4);
        asm volatile("" : "+r"(dv));
        if (wide) {   // O^T += V^T P^T: V with its rows for K, P from shared memory
          uint32_t dp = dq1 + g * (T::P >> 4);
          asm volatile("" : "+r"(dp));
#pragma unroll
          for (int k = 0; k < 8; ++k)
            umma_bf16(tm + COL_O + g * OST, UPPER | (dv + k * (2048 >> 4)), UPPER | (dp + (k >> 2) * (T::PCHUNK >> 4) + 2 * (k & 3)), ID_FEW | (1u << 15) | wide,
                      (!first || k > 0) ? 1u : 0u);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)   // 16 keys: 8 columns of P, two 8-key atoms of V
            umma_f16_ts(tm + COL_O + g * OST, tm + COL_S + g * 128 + 8 * k, UPPER | (dv + k * (2048 >> 4)), ID_O, (!first || k > 0) ? 1u : 0u);
        }
        fap_commit(&o_full[g]);
      };
      auto wide_of = [&](const ChunkPiece& p) { return p.kind == CHUNK_FEW ? (uint32_t)((p.tokens * a.G + 15) / 16 * 2) << 17 : 0u; };
      // the next piece; warp-uniform, and known to be
      auto fetch = [&](int& at, ChunkPiece& p) {
        const bool more = chunk_piece(a, list, begin, at, end, p);
        at = __shfl_sync(0xffffffffu, at, 0);
        p.n = __shfl_sync(0xffffffffu, p.n, 0);
        p.kind = __shfl_sync(0xffffffffu, p.kind, 0);
        p.tokens = __shfl_sync(0xffffffffu, p.tokens, 0);
        p.cnt0 = __shfl_sync(0xffffffffu, p.cnt0, 0);
        p.cnt1 = __shfl_sync(0xffffffffu, p.cnt1, 0);
        return __shfl_sync(0xffffffffu, (int)more, 0) != 0;
      };
      auto wait_k = [&](int t) { alive &= gemm_wait(smem_u32(&k_full[t % RK]), (t / RK) & 1, abortp); };
      auto wait_v = [&](int t) { alive &= gemm_wait(smem_u32(&v_full[t % RV]), (t / RV) & 1, abortp); };
      // the first scores of group g of piece p, whose key tiles begin at tile t and whose query tiles are number q0, q1
      auto open = [&](const ChunkPiece& p, int g, int t, int q0, int q1) {
        const bool pair = p.kind == CHUNK_PAIR;
        const int tile = pair ? g : 0, step = pair ? 0 : g;
        alive &= gemm_wait(smem_u32(&q_full[tile]), (tile ? q1 : q0) & 1, abortp);
        wait_k(t + step);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_one() && alive) {
          qk(g, tile, t + step, wide_of(p));
          if (!pair) fap_commit(&k_empty[(t + step) % RK]);                    // (of a pair, both tiles read the same keys)
          if (pair ? p.cnt(g) == 1 : step == p.n - 1) fap_commit(&q_empty[tile]);   // behind the last scores Q's place is free
        }
      };
      bool ahead[2] = {false, false};              // this piece's first scores of group g are issued already
      int at = begin;
      ChunkPiece p, next;
      bool more = fetch(at, next);
      while (more) {
        p = next;
        more = fetch(at, next);
        const int tn = ck + p.n;                   // the next piece's first key tile
        const bool pair = p.kind == CHUNK_PAIR;
        const int nq0 = cq[0] + (pair ? p.cnt0 > 0 : 1), nq1 = cq[1] + (pair && p.cnt1 > 0);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (p.cnt(g) > 0 && !ahead[g]) open(p, g, ck, cq[0], cq[1]);
          ahead[g] = false;
        }
        // the next piece's scores, while this one's last tiles and its O are worked on
        // (The second key tile's scores come behind the first's: the last ones give Q's place up.)
        auto go_on = [&](int g) {
          if (more && next.cnt(g) > 0 && (next.kind == CHUNK_PAIR || g == 0 || ahead[0])) {
            open(next, g, tn, nq0, nq1);
            ahead[g] = true;
          }
        };
        if (pair) {
          if (elect_one() && alive) fap_commit(&k_empty[ck % RK]);
          for (int j = 0; j < p.n; ++j) {
            const int t = ck + j;
            wait_v(t);
            if (!F8 && j + 1 < p.n) wait_k(t + 1);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int ng = p.cnt(g);
              if (j < ng) {
                alive &= gemm_wait(smem_u32(&p_full[g]), (c[g] + j) & 1, abortp);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if constexpr (F8) {   // (the next keys are being converted: the product does not wait for them)
                  if (elect_one() && alive) pv(g, t, j == 0, 0);
                  if (j + 1 < ng) {
                    wait_k(t + 1);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one() && alive) {
                      qk(g, g, t + 1, 0);
                      if (j + 2 == ng) fap_commit(&q_empty[g]);
                    }
                  }
                } else if (elect_one() && alive) {
                  pv(g, t, j == 0, 0);
                  if (j + 1 < ng) {
                    qk(g, g, t + 1, 0);
                    if (j + 2 == ng) fap_commit(&q_empty[g]);
                  }
                }
                // (the turned kind's P goes where Q1 is: not before this piece's last scores of tile 1 are on their way.  Where K has one place, the next piece's
                // first keys come behind this one's last.)
                if (j + 1 == ng && (!F8 || j + 1 == p.n) && (next.kind != CHUNK_FEW || g || j + 1 == p.n)) go_on(g);
              }
            }
            if (elect_one() && alive) {
              fap_commit(&v_empty[t % RV]);
              if (j + 1 < p.n) fap_commit(&k_empty[(t + 1) % RK]);
            }
          }
        } else {
          const uint32_t wide = wide_of(p);
          for (int j = 0; j < p.n; ++j) {
            const int t = ck + j, g = j & 1;
            wait_v(t);
            alive &= gemm_wait(smem_u32(&p_full[g]), (c[g] + (j >> 1)) & 1, abortp);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one() && alive) {
              pv(g, t, j < 2, 2 * wide);   // (P with the second halves of its weights)
              fap_commit(&v_empty[t % RV]);
              if (F8 && wide && j + 1 == p.n) fap_commit(&turn_free[few_pieces & 1]);
            }
            if (j + 2 < p.n) {
              wait_k(t + 2);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              if (elect_one() && alive) {
                qk(g, 0, t + 2, wide);
                fap_commit(&k_empty[(t + 2) % RK]);
                if (j + 3 == p.n) fap_commit(&q_empty[0]);
              }
            } else if (!(wide && next.kind == CHUNK_PAIR && g && j + 1 < p.n)) {   // (Q1 of a pair comes behind the last product that reads P)
              go_on(g);
            }
          }
        }
        c[0] += p.cnt0; c[1] += p.cnt1; ck = tn;
        cq[0] = nq0; cq[1] = nq1;
        few_pieces += p.kind == CHUNK_FEW;
      }
    }
    // ------------------------------------------------------------------------------------------------ scales of 8-bit pages
    if (F8 && warp == 10) {
      bool alive = true;
      int c[2] = {0, 0};
      int at = begin;
      ChunkPiece p;
      while (alive && chunk_piece(a, list, begin, at, end, p)) {
        const int32_t* const pages = a.table + (size_t)p.request * a.blocks;
        const int last_page = (p.pos0 + p.tokens - 1) / kStepPage;
        int first = 2 * p.k0;
        float to_log2, value;   // of 32 pages from `first` on, a lane each
        auto read = [&]() {
          const size_t e = (size_t)__ldg(pages + min(first + lane, last_page)) * a.Hkv + p.head;
          to_log2 = __ldg(a.k_scales + e) * a.scale_log2e;
          value = __ldg(a.v_scales + e);
        };
        read();
        for (int j = 0; alive && j < p.n; ++j) {
          if (2 * (p.k0 + j) >= first + 32) {
            first += 32;
            read();
          }
          const int h = lane - (2 * (p.k0 + j) - first);   // 0, 1: the tile's pages
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (p.kind == CHUNK_PAIR ? j >= p.cnt(g) : (j & 1) != g) continue;
            const int n = c[g]++, i = n % kChunkScales;
            if (!(alive = gemm_wait_warp(smem_u32(&sc_empty[g][i]), ((n / kChunkScales) & 1) ^ 1, abortp))) break;
            if (h == 0 || h == 1) {
              float* const to = sc[g][i] + h;
              to[0] = to_log2;
              to[2] = log2f(value);
              to[4] = 1.f / value;
              to[6] = value;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sc_full[g][i]);
          }
        }
      }
    }
    // ------------------------------------------------------------------------------------------------ 8-bit pages to bf16 tiles
    // 16 codes of a row a thread at a time: 16 bytes read, two pieces of 16 bytes written, whose places in the swizzled tile are other banks for each of eight lanes
    // (at head size 128 a row's second 64 features lie 16 KB behind: half of the lanes write their second piece first).
    if (F8 && warp >= 12) {
      const int ct = tid - 384;
      constexpr int ROW = D / 16, PIECES = 64 * ROW / 128;   // 16-byte pieces of a row; of a page, a thread
      const int c16 = ct % ROW, row0 = ct / ROW;
      const int f0 = 2 * c16 + (D == 128 && c16 >= 4 ? 1 : 0);
      bool alive = true;
      int ck = 0, cp = 0;
      int at = begin;
      ChunkPiece p;
      while (alive && chunk_piece(a, list, begin, at, end, p)) {
        for (int j = 0; alive && j < p.n; ++j, ++ck) {
#pragma unroll 1
          for (int kv = 0; alive && kv < 2; ++kv) {
            const int i = kv ? ck % RV : ck % RK, ph = kv ? (ck / RV) & 1 : (ck / RK) & 1;
            uint64_t* const full = kv ? &v_full[i] : &k_full[i];
            const uint32_t tile = kv ? smV + i * T::TILE : smK + i * T::TILE;
#pragma unroll 1
            for (int r = 0; r < 2; ++r, ++cp) {
              const int q = cp % T::PAGES;
              if (!(alive = gemm_wait_warp(smem_u32(&c_full[q]), (cp / T::PAGES) & 1, abortp))) break;
              uint4 w[PIECES];
#pragma unroll
              for (int e = 0; e < PIECES; ++e) w[e] = lds128(smC + q * T::PAGE + (e * 128 + ct) * 16);
              __syncwarp();
              if (lane == 0) mbar_arrive(&c_empty[q]);
              if (r == 0 && !(alive = gemm_wait_warp(kv ? smem_u32(&v_empty[i]) : smem_u32(&k_empty[i]), ph ^ 1, abortp))) break;
#pragma unroll
              for (int e = 0; e < PIECES; ++e) {
                const int row = r * 64 + row0 + e * (128 / ROW);
                uint4 lo = make_uint4(chunk_widen(w[e].x, 0x1404), chunk_widen(w[e].x, 0x3424), chunk_widen(w[e].y, 0x1404), chunk_widen(w[e].y, 0x3424));
                uint4 hi = make_uint4(chunk_widen(w[e].z, 0x1404), chunk_widen(w[e].z, 0x3424), chunk_widen(w[e].w, 0x1404), chunk_widen(w[e].w, 0x3424));
                if (f0 & 1) { const uint4 t = lo; lo = hi; hi = t; }
                const uint32_t dst = tile + (f0 >> 3) * 16384 + row * 128;
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + (((f0 & 7) ^ (row & 7)) << 4)), "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w) : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst + ((((f0 ^ 1) & 7) ^ (row & 7)) << 4)), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w) : "memory");
              }
            }
            if (!alive) break;
            fence_proxy_async();   // generic-proxy stores -> the tensor core's async proxy
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
          }
        }
      }
    }
    // ------------------------------------------------------------------------------------------------ rows behind the last request's
    if (warp == T::W_REST && a.rest) {
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

template <int D, bool F8 = false>
static cudaError_t launch_chunk(const CUtensorMap (&m)[4], const ChunkArgs& a, cudaStream_t st) {
  using T = ChunkTile<D, F8>;
  static std::atomic<unsigned long long> served{0};
  const cudaError_t set = once_per_device(served, [] {
    cudaFuncAttributes at;
    const cudaError_t e = cudaFuncGetAttributes(&at, chunk_attn_kernel<D, F8>);
    if (e != cudaSuccess) return e;
    // the warps' register shares must fit what the block is launched with, or they would wait for registers for good
    if (at.numRegs * T::THREADS < 8 * 32 * T::REGS_SOFTMAX + (T::THREADS - 256) * T::REGS_REST) return cudaErrorInvalidConfiguration;
    return cudaFuncSetAttribute(chunk_attn_kernel<D, F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
  });
  if (set != cudaSuccess) return set;
  count_launch();
  return launch_pdl(chunk_attn_kernel<D, F8>, dim3((unsigned)(num_sms() < kStepMaxCtas ? num_sms() : kStepMaxCtas)), dim3(T::THREADS), T::SMEM, st, m[0], m[1], m[2], m[3], a);
}

static size_t chunk_workspace_bytes(int D) { return kStepMaxCtas * 4 + (size_t)2 * kStepMaxCtas * (D == 128 ? kChunkRecord<128> : kChunkRecord<64>) * 4; }
// the common part: q's maps, the plan's arrays
template <bool F8>
static int chunk_common(ChunkArgs& a, CUtensorMap* maps, void* out, const pie_head_rows* q, const int32_t* plan, const pie_step_dims* d, int D, float scale, int rest,
                        void* workspace, size_t workspace_bytes) {
  if ((D != 64 && D != 128) || !(scale > 0.f) || scale > 3.4028234e38f / 1.5f || q->stride_h % 8 || q->stride_l % 8 || (d->rows > 1 && q->stride_l <= 0) ||
      (d->Hq > 1 && q->stride_h <= 0))
    return PIE_EINVAL_SHAPE;
  for (const void* p : {(const void*)out, q->p, (const void*)plan, (const void*)workspace})
    if (reinterpret_cast<uintptr_t>(p) & 15) return PIE_EALIGN;
  if (!workspace || workspace_bytes < chunk_workspace_bytes(D)) return PIE_EWORKSPACE;
  const StepLayout l = step_layout(*d);
  a = {};
  a.out = (uint16_t*)out; a.Hq = d->Hq; a.Hkv = d->Hkv; a.G = d->Hq / d->Hkv; a.tile_tokens = l.tile_tokens; a.rows = d->rows; a.requests = d->requests;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.ranges = plan + l.ranges; a.table = plan + l.block_table; a.row_starts = plan + l.row_starts;
  a.pieces = reinterpret_cast<const StepPiece*>(plan + l.pieces);
  a.blocks = d->blocks; a.rest = rest;
  a.count = (unsigned int*)workspace;
  a.part = (float*)((uint8_t*)workspace + kStepMaxCtas * 4);
  const GemmEncodeFn fn = gemm_encode_fn();
  if (!fn) return PIE_ECUDA;
  const cuuint32_t one[4] = {1, 1, 1, 1};
  // a query tile, and one of the turned kind: 64 features of G heads of their tokens
  a.few_tokens = (D == 128 ? ChunkTile<128, F8>::FEW : ChunkTile<64, F8>::FEW) / a.G;
  for (int i = 0; i < 2; ++i) {
    const long long head = (d->Hq > 1 ? q->stride_h : D) * 2, row = (d->rows > 1 ? q->stride_l : (long long)d->Hq * D) * 2;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)d->Hq, (cuuint64_t)d->rows}, strides[2] = {(cuuint64_t)head, (cuuint64_t)row};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)(i && a.few_tokens ? a.few_tokens : a.tile_tokens)};
    if (fn(&maps[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q->p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return PIE_EUNSUPPORTED;
  }
  return PIE_OK;
}

}  // namespace pie

extern "C" {

using namespace pie;

size_t pie_chunk_attn_workspace_bytes(const pie_step_dims* d, int D) {
  if (step_dims_status(d) || (D != 64 && D != 128)) return 0;
  return chunk_workspace_bytes(D);
}

int pie_chunk_attn(void* out, const pie_head_rows* q, const void* kpool, const void* vpool, const pie_kv_layout* kv, const int32_t* plan, const pie_step_dims* d, int D,
                   float scale, int rest, void* workspace, size_t workspace_bytes, void* stream) {
  if (int s = step_dims_status(d)) return s;
  if (!out || !q || !q->p || !kpool || !vpool || !kv || !plan) return PIE_ENULL;
  if (kv->tok_stride <= 0 || kv->tok_stride % 8 || kv->head_stride % 8 || (d->Hkv > 1 && kv->head_stride <= 0)) return PIE_EINVAL_SHAPE;
  ChunkArgs a;
  CUtensorMap maps[4];
  if (int s = chunk_common<false>(a, maps, out, q, plan, d, D, scale, rest, workspace, workspace_bytes)) return s;
  for (const void* p : {kpool, vpool})
    if (reinterpret_cast<uintptr_t>(p) & 15) return PIE_EALIGN;
  const GemmEncodeFn fn = gemm_encode_fn();
  const cuuint32_t one[4] = {1, 1, 1, 1};
  for (int i = 0; i < 2; ++i) {   // a page of one head: 64 features of its 64 slots
    const long long tok = kv->tok_stride * 2, head = d->Hkv > 1 ? kv->head_stride * 2 : tok;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)kStepPage, (cuuint64_t)d->Hkv, (cuuint64_t)d->pages};
    const cuuint64_t strides[3] = {(cuuint64_t)tok, (cuuint64_t)head, (cuuint64_t)(kStepPage * tok)};
    const cuuint32_t box[4] = {64, 64, 1, 1};
    if (fn(&maps[2 + i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(i ? vpool : kpool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, D == 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)   // (256 bytes at head size 64 are two heads: half as much again was read from HBM)
      return PIE_EUNSUPPORTED;
  }
  return status_of(D == 128 ? launch_chunk<128>(maps, a, (cudaStream_t)stream) : launch_chunk<64>(maps, a, (cudaStream_t)stream));
}

int pie_chunk_attn_fp8(void* out, const pie_head_rows* q, const uint8_t* kpool, const float* k_scales, const uint8_t* vpool, const float* v_scales, const int32_t* plan,
                       const pie_step_dims* d, int D, float scale, int rest, void* workspace, size_t workspace_bytes, void* stream) {
  if (int s = step_dims_status(d)) return s;
  if (!out || !q || !q->p || !kpool || !k_scales || !vpool || !v_scales || !plan) return PIE_ENULL;
  ChunkArgs a;
  CUtensorMap maps[4];
  if (int s = chunk_common<true>(a, maps, out, q, plan, d, D, scale, rest, workspace, workspace_bytes)) return s;
  for (const void* p : {(const void*)kpool, (const void*)vpool})
    if (reinterpret_cast<uintptr_t>(p) & 15) return PIE_EALIGN;
  maps[2] = maps[3] = maps[0];   // (its keys and values come by address)
  a.k8 = kpool; a.v8 = vpool; a.k_scales = k_scales; a.v_scales = v_scales;
  return status_of(D == 128 ? launch_chunk<128, true>(maps, a, (cudaStream_t)stream) : launch_chunk<64, true>(maps, a, (cudaStream_t)stream));
}

}  // extern "C"
