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
// Device time in a row of such calls, inputs not in L2, 32 query / 8 kv heads: D 128, 2048 tokens behind 15000 468 us (1150 TFLOP/s, of cuBLAS's 1638 in a burst; 490 to 508 in a long run, at a lower clock; the tensor pipe is
// busy for 54 % of it, as in the prompt's kernel one tile's softmax is covered by the other's products in part); 16 answers with up to five drafted tokens over 4000 keys 51.6 (4.4 TB/s),
// 40 over 12000 309 (6.4 TB/s), one with four over 9000 26.3; D 64, three portions of 700 tokens beside 29 answers over 1500 keys 83.9, 40 answers over 12000 220 (4.5 TB/s).  Short
// steps pay 4 us from the launch to the first scores, some 3 at each turn from one piece to the next and 5 at the end: results, one counter, the last CTA's sums.
// Pages of 8 bits (F8): the turned kind's operands are the codes as they lie (below); of requests of more rows the pages are brought to 16 bits by a launch in front (chunk_widen_kernel).
// us, and over 16-bit pages in the same run: 40 answers with up to five drafts over 6000 keys 122 (4.2 TB/s), 175; without drafts 107 (4.7 TB/s), 166; over 12000 keys 197, 314; one with four over
// 9000 25.8, 26.3; D 64, 40 over 12000 181, 222.  Where prompts take part nothing is won: three portions beside 29 answers over 1500 keys 99.5, 92 (D 64: 119, 111), 2048 tokens behind 15000 502, 469
// (557 to 568 in a long run).
#include <type_traits>

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
  // 8-bit pages: their scales [pages, Hkv], and queries as they lie (elements between rows, between heads)
  const float *k_scales, *v_scales;
  const int32_t* contexts;
  int Hkv;
  const uint16_t* q;
  long long q_row, q_head;
};
template <int D>
constexpr int kChunkRecord = 256 * D + 512;   // floats: results, [64 rows][D] of the turned kind, [D / 4][256 rows][4] of the others; [256] maxima and sums
constexpr int kChunkFew = 64;                 // rows of an item of the turned kind, at most (ChunkTile::FEW)
constexpr int kChunkList = 32;                // pieces held in shared memory; a CTA that has more reads them where they are

template <int D, bool F8 = false>
struct ChunkTile {
  static constexpr int CH = D / 64, TILE = 128 * D * 2;          // 64-feature chunks of a row, bytes of 128 rows
  static constexpr int RING = D == 64 ? 4 : 2;                   // tiles of K, and of V: 64 KB of each
  static constexpr int FEW = F8 ? 32 : D == 64 ? 64 : 48;        // rows of an item of the turned kind, at most: as shared memory has room for their weights (8-bit pages: as tensor memory has for four tiles' scores)
  static constexpr int PCHUNK = 2 * FEW * 128;                   // bytes of 64 keys of a group's P of the turned kind: eight rows' first halves, their second halves, ...
  static constexpr int P = F8 ? 3 * FEW * 128 : 2 * PCHUNK;      // (8-bit pages: three numbers a weight, a byte each)
  static constexpr int Q1 = TILE > 2 * P ? TILE : 2 * P;         // the second query tile; the turned kind's P
  static constexpr int PLACES = 2 * RING;                        // 8-bit pages, turned kind: a key tile's codes of K and of V take one tile's place
  static constexpr int QF = 2 * FEW * D;                         // and the queries of a piece, as two codes a feature; two pieces' are held
  static constexpr int SMEM = 1024 + TILE + Q1 + 2 * RING * TILE + (F8 ? 2 * QF : 0);
  static constexpr int THREADS = 384;
};
constexpr int kChunkScales = 8;               // 8-bit pages: key tiles whose scales are held

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

struct ChunkMaps8 { CUtensorMap k, v; };   // of the codes, a page of a head
struct ChunkNone {};
// two codes as fp16, exactly; numbers to codes
__device__ __forceinline__ uint32_t chunk_f16(uint32_t two) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((uint16_t)two));
  return d;
}
__device__ __forceinline__ void chunk_f32(uint32_t f16x2, float& lo, float& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(lo), "=f"(hi) : "r"(f16x2));
}
__device__ __forceinline__ uint32_t chunk_codes4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return lo | ((uint32_t)hi << 16);
}
// D[128 x N] (+)= A B of 8-bit numbers, both from shared memory
__device__ __forceinline__ void chunk_mma_f8(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(accum) : "memory");
}
__device__ __forceinline__ void chunk_ld8(uint32_t taddr, float* v) {   // not waited for
  uint32_t* const u = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
               : "r"(taddr) : "memory");
}
__device__ __forceinline__ void chunk_st8(uint32_t taddr, const float* v) {
  const uint32_t* const u = reinterpret_cast<const uint32_t*>(v);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ uint32_t chunk_pack_f16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Two fp16 as three pairs of e5m2 numbers, each in a half's upper byte, whose sums they are: of eleven bits the first takes three, and what it leaves, which has a sign, each of the others
// four.  (Below 2^-5 the lowest bits lie below e5m2's lowest, 2^-16.)  e5m2 is fp16 without its lowest eight bits, so that a rounding is an addition; no half is near the largest.
__device__ __forceinline__ void chunk_thirds(uint32_t x, uint32_t (&to)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    to[i] = (x + 0x00800080u) & 0xff00ff00u;
    if (i < 2) asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(x) : "r"(x), "r"(to[i]));
  }
}
// whether a round is over; all of a warp's lanes are told the same
__device__ __forceinline__ bool chunk_ready(const uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, ok);
}
// where 16 bytes of a row of a page lie in its place in shared memory
template <int D>
__device__ __forceinline__ uint32_t chunk_code_at(int row, int c16) {
  return D == 128 ? row * 128 + ((c16 ^ (row & 7)) << 4) : row * 64 + ((c16 ^ ((row >> 1) & 3)) << 4);
}

template <int D, bool F8>
__global__ void __launch_bounds__(ChunkTile<D, F8>::THREADS, 1)
chunk_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_few, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ typename std::conditional<F8, ChunkMaps8, ChunkNone>::type codes8,
                  const __grid_constant__ ChunkArgs a) {
  using T = ChunkTile<D, F8>;
  constexpr int RING = T::RING;
  constexpr uint32_t ID_S = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t ID_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
  constexpr uint32_t ID_FEW = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);   // | N
  constexpr int COL_S = 0, COL_O = 256, OST = 128;   // + g * 128, + g * OST
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[RING], k_empty[RING], v_full[RING], v_empty[RING], s_full[2], p_full[2], o_full[2];
  __shared__ __align__(16) int4 list[3 * kChunkList];
  // 8-bit pages, turned kind: places of its key tiles, their scales, the queries of a piece (two in turn), its last product (in turn), behind which P's place is free, four tiles' scores, and weights and
  // products of either group, whose tiles are every other one
  __shared__ __align__(8) uint64_t f_full[F8 ? T::PLACES : 1], f_empty[F8 ? T::PLACES : 1], sc_full[F8 ? kChunkScales : 1], sc_empty[F8 ? kChunkScales : 1], qf_full[2], qf_empty[2], turn_free[2], fs_full[4], fp_full[2], fo_full[2];
  __shared__ __align__(16) float4 sc[F8 ? kChunkScales : 1][2];   // of either page of a tile: scores to log2 units, log2 of the values' scale, its reciprocal
  __shared__ __align__(16) float q_scale[2][F8 ? T::FEW : 4];
  __shared__ __align__(16) ChunkFew few;
  __shared__ float2 ml[2][128];           // a row's maximum and sum: of the two groups of a tile, of the rows of a cut item
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, last_flag;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  // (The turned kind's P lies where Q1 does.  Its V^T has 128 rows whatever the head size: at 64 the upper ones are what lies 16 KB behind, so V does not lie last.)
  const uint32_t smV = base, smK = smV + RING * T::TILE, smQ = smK + RING * T::TILE, smQ1 = smQ + T::TILE, smF = smQ1 + T::Q1;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < RING; ++i) {
      mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
    }
    if (F8) {
      for (int i = 0; i < T::PLACES; ++i) { mbar_init(&f_full[i], 1); mbar_init(&f_empty[i], 1); }
      for (int i = 0; i < kChunkScales; ++i) { mbar_init(&sc_full[i], 1); mbar_init(&sc_empty[i], 4); }
      for (int i = 0; i < 2; ++i) { mbar_init(&qf_full[i], 1); mbar_init(&qf_empty[i], 9); mbar_init(&turn_free[i], 1); mbar_init(&fp_full[i], 4); mbar_init(&fo_full[i], 1); }
      for (int i = 0; i < 4; ++i) mbar_init(&fs_full[i], 1);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 8 && lane < 4) tma_prefetch_desc(lane == 0 ? &map_q : lane == 1 ? &map_few : lane == 2 ? &map_k : &map_v);
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
    asm volatile("bar.sync 4, 352;" ::: "memory");
    if (end - begin > 1) asm volatile("bar.arrive 5, 384;" ::: "memory");
  }

  // All barriers are counted over the CTA's pieces: a role keeps the number of key tiles (of its group, of K and V) before its piece.
  // Registers: 384 threads x 168 at launch = 64512; 8 warps of 216 and 4 of 64 are 63488.
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------------------------------------------ softmax of group g
    const int g = warp >> 2, quad = warp & 3, r = quad * 32 + lane, tok = r / a.G;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t tS = tmem + COL_S + g * 128 + lanes, tO = tmem + COL_O + lanes;
    int c[2] = {0, 0}, cv = 0;     // key tiles of either group, tiles of V, before this piece
    int cf = 0, few_pieces = 0;    // 8-bit pages: key tiles and pieces of the turned kind before this one, which the other counts leave out
    bool alive = true;
    int at = begin;
    ChunkPiece p;
    // values behind the item's last key may be anything: this thread's row of the key tile they lie in
    auto clear_tail = [&](int step, int tail) {
      const int v = cv + step;
      alive = alive && gemm_wait_warp(smem_u32(&v_full[v % RING]), (v / RING) & 1, abortp);
      if (alive && r >= tail)
#pragma unroll
        for (int q = 0; q < 8 * T::CH; ++q)
          asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(smV + (v % RING) * T::TILE + (q >> 3) * 16384 + r * 128 + (q & 7) * 16), "r"(0) : "memory");
      fence_proxy_async();
    };
    // Registers are short where a thread holds a row of scores: the loops keep a few numbers, and the piece is read again behind them.
    auto read_again = [&]() {
      const volatile int* const e = reinterpret_cast<const volatile int*>(chunk_words(a, list, begin, at - 1));
      p.row0 = e[0]; p.pos0 = e[1]; p.tokens = e[2]; p.head = e[4]; p.first = e[7]; p.pieces = e[8];
    };
    while (chunk_piece(a, list, begin, at, end, p)) {
      const int keys = p.pos0 + p.tokens, tail = keys & 127, tail_step = tail ? (keys - 1) / 128 - p.k0 : -1, cnt = p.cnt(g);
      if (F8 && p.kind == CHUNK_FEW) {
        // ---------------------------------------------------------------------------------- 8-bit pages: a key a lane, a row a column
        // As below, with other operands, and bound by the stream of pages, half as long.  The codes of K and V are the MMAs' as they lie, and all else is made to suit them: a query, brought to
        // 2^7 .. 2^8 by a power of two for each row, is the sum of two e4m3 numbers (its first four and its last four bits; what is 2^-17 of the row's largest is lost), a weight, as fp16, of
        // three e5m2 numbers, each with columns of its own, that are added up as fp32.  The MMA with its 128 keys or features by 16 to 96 columns is a hundred cycles or two; what it costs
        // to widen the codes instead was 2.9 us a key tile by way of shared memory and 2.2 in registers (mma.sync, 24 rows), where the stream takes 0.75.
        // A row's reference is that of its weights times their pages' scale of V, so that its results are in the units of the largest of those, whatever scales the pages have; its sum is rid of
        // the scale again.  The CTA's key tiles of this kind go to the groups in turn, and four tiles' scores are under way at a time, of the next piece too, so that a group never waits for
        // the products of its last tile (40 answers with up to five drafts over 6000 keys: two tiles' scores, rows in fours 184 us; four tiles', rows in eights
        // without a branch 143; two numbers an instruction, and P in words, turned around among four lanes, in place of bytes 125).
        if constexpr (F8) {
          const int rows = p.tokens * a.G, which = few_pieces & 1, half = quad >> 1, own = (g ^ cf) & 1;   // the group's first tile
          const int cnt_own = (p.n + 1 - own) / 2, cnt_other = p.n - cnt_own;
          const int beyond = p.k0 * 128 + r - p.pos0, edge_step = (p.pos0 + 1) / 128 - p.k0;   // the first key tile with a key that some row must not see
          const uint32_t turn1 = lane & 1 ? 0x3715 : 0x6240, turn2 = lane & 2 ? 0x3276 : 0x5410;
          uint32_t sp[2];   // this lane's four keys in P's rows lane % 4, and four on
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int row = 4 * k + (lane & 3);
            sp[k] = smQ1 + g * T::P + row * 128 + (((r >> 4) ^ row) << 4) + (r & 12);
          }
          alive = alive && gemm_wait_warp(smem_u32(&qf_full[which]), (few_pieces >> 1) & 1, abortp);   // (for the queries' scales)
          auto weights = [&](auto blocks) {
            constexpr int N = 8 * decltype(blocks)::value;
            float l[32];
#pragma unroll
            for (int n = 0; n < 32; ++n) l[n] = 0.f;
            for (int i = 0; i < cnt_own; ++i) {
              const int step = 2 * i + own, tile = cf + step, is = tile % kChunkScales;
              alive = alive && gemm_wait_warp(smem_u32(&sc_full[is]), (tile / kChunkScales) & 1, abortp);
              const float4 of = sc[is][half];
              __syncwarp();
              if (lane == 0) mbar_arrive(&sc_empty[is]);
              alive = alive && gemm_wait_warp(smem_u32(&fs_full[tile & 3]), (tile >> 2) & 1, abortp);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              float v[2 * N], s[N];   // (two at a time where that is one instruction)
#pragma unroll
              for (int b = 0; b < N / 8; ++b) chunk_ld16(tS + 32 * (tile & 2) + 16 * b, v + 16 * b);
              tmem_ld_wait();
#pragma unroll
              for (int n = 0; n < N; n += 4) {
                const float4 q = *reinterpret_cast<const float4*>(&q_scale[which][n]);
                const float f[4] = {q.x, q.y, q.z, q.w}, *const hi = v + 2 * n - n % 8;
#pragma unroll
                for (int k = 0; k < 4; k += 2)
                  f2_unpack(f2_fma(f2_add(f2_pack(hi[k], hi[k + 1]), f2_pack(hi[8 + k], hi[9 + k])), f2_mul(f2_pack(f[k], f[k + 1]), f2_pack(of.x, of.x)), f2_pack(of.y, of.y)), s[n + k], s[n + k + 1]);
              }
              if (step >= edge_step) {
                const int cut = (beyond + step * 128) * a.G;
#pragma unroll
                for (int n = 0; n < N; ++n)
                  if (n < cut) s[n] = -INFINITY;
              }
              bool over = i == 0;
              if (i > 0) {
                float mx = -INFINITY;
#pragma unroll
                for (int n = 0; n < N; n += 4) {
                  const float4 less = *reinterpret_cast<const float4*>(&few.less[g][n]);
                  f2_unpack(f2_add(f2_pack(s[n], s[n + 1]), f2_pack(less.x, less.y)), s[n], s[n + 1]);
                  f2_unpack(f2_add(f2_pack(s[n + 2], s[n + 3]), f2_pack(less.z, less.w)), s[n + 2], s[n + 3]);
                  mx = fmaxf(fmaxf(mx, fmaxf(s[n], s[n + 1])), fmaxf(s[n + 2], s[n + 3]));
                }
                over = mx > 15.f;
                // behind the product before this one P's place is free, and O holds the tiles so far
                alive = alive && gemm_wait_warp(smem_u32(&fo_full[g]), ((tile >> 1) - 1) & 1, abortp);
              }
              // The reference of a row, four times the largest weight that it was made from, moves where a weight exceeds it 16 times.  (At once the largest: scores of 2.9 log2 units' deviation
              // move some of 24 rows' in every fifth tile; so in one of twenty.)
              if (chunk_group_any(g, over)) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                int mine = 0;
#pragma unroll
                for (int n = 0; n < N; ++n) {
                  if (i > 0) s[n] -= few.less[g][n];
                  const int x = __reduce_max_sync(0xffffffffu, chunk_order(s[n]));
                  if (lane == n) mine = x;
                }
                few.best[g][quad][lane] = mine;
                chunk_group_sync(g);
                if (quad == 0 && lane < N) {
                  const float was = i == 0 ? -INFINITY : few.m[g][lane];
                  const float now = chunk_unorder(max(max(few.best[g][0][lane], few.best[g][1][lane]), max(few.best[g][2][lane], few.best[g][3][lane])));
                  const bool move = i == 0 || now > was + 4.f;
                  const float m = move ? now + 2.f : was;
                  few.factor[g][lane] = !move ? 1.f : was == -INFINITY ? 0.f : fap_exp2(was - m);
                  few.m[g][lane] = m;
                  few.less[g][lane] = m == -INFINITY ? 0.f : 11.f - m;   // weights of up to 2^15
                }
                chunk_group_sync(g);
#pragma unroll
                for (int n = 0; n < N; ++n) s[n] += few.less[g][n];
                if (i > 0) {
#pragma unroll
                  for (int b = 0; b < N / 8; ++b) {
                    float f[8];
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                      f[n] = few.factor[g][8 * b + n];
                      l[8 * b + n] *= f[n];
                    }
#pragma unroll 1
                    for (int k = 0; k < 3; ++k) {
                      float o[8];
                      chunk_ld8(tO + g * OST + 24 * b + 8 * k, o);
                      tmem_ld_wait();
#pragma unroll
                      for (int n = 0; n < 8; ++n) o[n] *= f[n];
                      chunk_st8(tO + g * OST + 24 * b + 8 * k, o);
                    }
                  }
                  tmem_st_wait();
                }
              }
#pragma unroll
              for (int n = 0; n < N; n += 4) {
                uint32_t c3[2][3];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  float* const ln = l + n + 2 * k;
                  const float e0 = fap_exp2(s[n + 2 * k]), e1 = fap_exp2(s[n + 2 * k + 1]);
                  f2_unpack(f2_fma(f2_pack(e0, e1), f2_pack(of.z, of.z), f2_pack(ln[0], ln[1])), ln[0], ln[1]);
                  chunk_thirds(chunk_pack_f16(e0, e1), c3[k]);
                }
                // four rows of a key turned into four keys of a row, among four lanes
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                  uint32_t x = __byte_perm(c3[0][q], c3[1][q], 0x7531);
                  x = __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 1), turn1);
                  x = __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 2), turn2);
                  asm volatile("st.shared.u32 [%0], %1;" ::"r"(sp[n / 4 & 1] + (24 * (n / 8) + 8 * q) * 128), "r"(x) : "memory");
                }
              }
              if (step == tail_step) {   // values behind the item's last key
                alive = alive && gemm_wait_warp(smem_u32(&f_full[tile % T::PLACES]), (tile / T::PLACES) & 1, abortp);
                if (alive && r >= tail)
#pragma unroll
                  for (int q = 0; q < D / 16; ++q)
                    asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(smV + tile % T::PLACES * T::TILE + (128 + r) * D + 16 * q), "r"(0) : "memory");
              }
              fence_proxy_async();
              asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
              __syncwarp();
              if (lane == 0) mbar_arrive(&fp_full[g]);
            }
            // a row's sum over the warp's lanes: half of the columns a step, until a lane has one
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
              for (int k = 0; k < o; ++k) {
                const float give = lane & o ? l[k] : l[k + o], keep = lane & o ? l[k + o] : l[k];
                l[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
              }
            few.sum[g][quad][lane] = l[0];
          };
          switch ((rows - 1) / 8) {   // (rows behind the last are worked on with those beside them: their scores are 0)
            case 0: weights(std::integral_constant<int, 1>()); break;
            case 1: weights(std::integral_constant<int, 2>()); break;
            case 2: weights(std::integral_constant<int, 3>()); break;
            default: weights(std::integral_constant<int, 4>());
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&qf_empty[which]);
          const int cnt0 = g ? cnt_other : cnt_own, cnt1 = g ? cnt_own : cnt_other;
          read_again();
          const bool whole = p.pieces == 1;
          float* const rec = a.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == p.first)) * kChunkRecord<D>;
          if (cnt_own > 0) alive = alive && gemm_wait_warp(smem_u32(&fo_full[g]), ((cf + 2 * cnt_own - 2 + own) >> 1) & 1, abortp);
          cf += p.n; ++few_pieces;
          chunk_sync();     // (the other group has waited for its own)
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (tid < rows) {
            const float m0 = cnt0 > 0 ? few.m[0][tid] : -INFINITY, m1 = cnt1 > 0 ? few.m[1][tid] : -INFINITY, m = fmaxf(m0, m1);
            const float f0 = m0 == -INFINITY ? 0.f : fap_exp2(m0 - m), f1 = m1 == -INFINITY ? 0.f : fap_exp2(m1 - m);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if (cnt0 > 0) sum = fmaf(few.sum[0][w][tid], f0, sum);
              if (cnt1 > 0) sum = fmaf(few.sum[1][w][tid], f1, sum);
            }
            const float inv = whole ? 1.f / sum : 1.f;   // (weights and sums are 2^11 times too large)
            few.share[tid] = make_float2(f0 * inv, f1 * inv);
            const int t = tid / a.G;
            few.row[tid] = (p.row0 + t) * a.Hq + p.head * a.G + tid - t * a.G;
            if (!whole) __stcg(reinterpret_cast<float2*>(rec + 256 * D + 2 * tid), make_float2(m, sum));
          }
          chunk_sync();
          if (alive && (D == 128 || quad < 2)) {   // (head size 64: nothing in the upper lanes)
#pragma unroll 1
            for (int n0 = 8 * g; n0 < rows; n0 += 16) {
              float v[8];
#pragma unroll
              for (int n = 0; n < 8; ++n) v[n] = 0.f;
#pragma unroll 1
              for (int h = cnt0 > 0 ? 0 : 1; h < (cnt1 > 0 ? 2 : 1); ++h) {
                float o[24];
#pragma unroll
                for (int k = 0; k < 3; ++k) chunk_ld8(tO + h * OST + 3 * n0 + 8 * k, o + 8 * k);
                tmem_ld_wait();
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                  const float2 f = few.share[n0 + n];
                  v[n] = fmaf(o[n] + o[8 + n] + o[16 + n], h ? f.y : f.x, v[n]);
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
        }
      } else if (!F8 && p.kind == CHUNK_FEW) {
        if constexpr (!F8) {
        // ---------------------------------------------------------------------------------- a key a lane, a row a column
        const int rows = p.tokens * a.G;
        const int beyond = p.k0 * 128 + r - p.pos0, edge_step = (p.pos0 + 1) / 128 - p.k0;   // the first key tile with a key that some row must not see
        const uint32_t sp = smQ1 + g * T::P + (r >> 6) * T::PCHUNK + (r & 7) * 2;
        const int chunk16 = (r & 63) >> 3;
        float l[kChunkFew];
#pragma unroll
        for (int n = 0; n < kChunkFew; ++n) l[n] = 0.f;
        for (int i = 0; i < cnt; ++i) {
          const int step = 2 * i + g;
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
              s[n] = fap_exp2(fmaf(s[n], a.scale_log2e, less.x));
              s[n + 1] = fap_exp2(fmaf(s[n + 1], a.scale_log2e, less.y));
              s[n + 2] = fap_exp2(fmaf(s[n + 2], a.scale_log2e, less.z));
              s[n + 3] = fap_exp2(fmaf(s[n + 3], a.scale_log2e, less.w));
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
          if (i > 0 && rows > 32) {
            load(1);
            over = weigh(1) > 256.f;
          }
          load(0);
          if (i > 0) over = weigh(0) > 256.f || over;
          // the reference of a row moves where a score exceeds it by 8 (log2 units: a weight of 256): same sums, and mostly the lanes need not know of one another
          if (chunk_group_any(g, over)) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
              if (32 * half < rows) {
                if (half || i > 0) load(half);
                int mine = 0;
#pragma unroll
                for (int n = 0; n < 32; ++n) {
                  if (32 * half + n >= rows) break;
                  const int v = __reduce_max_sync(0xffffffffu, chunk_order(s[n]));
                  if (lane == n) mine = v;
                }
                few.best[g][quad][32 * half + lane] = mine;
              }
            chunk_group_sync(g);
            if (quad == 0)
              for (int n = lane; n < rows; n += 32) {
                const float was = i == 0 ? -INFINITY : few.m[g][n];
                const float now = chunk_unorder(max(max(few.best[g][0][n], few.best[g][1][n]), max(few.best[g][2][n], few.best[g][3][n]))) * a.scale_log2e;
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
            if (rows > 32 || i > 0) load(0);
            weigh(0);
          }
#pragma unroll
          for (int half = 0; half < 2; ++half)
            if (32 * half < rows) {
              if (half) {
                load(1);
                weigh(1);
              }
#pragma unroll
              for (int n = 0; n < 32; n += 4) {
                if (32 * half + n >= T::FEW || 32 * half + n >= rows) break;
                l[32 * half + n] += s[n]; l[32 * half + n + 1] += s[n + 1]; l[32 * half + n + 2] += s[n + 2]; l[32 * half + n + 3] += s[n + 3];
                const uint32_t w01 = pack_bf16(s[n], s[n + 1]), w23 = pack_bf16(s[n + 2], s[n + 3]);
                const int row = 2 * (32 * half + n) - n % 8;
                put(row, w01, w23);
                put(row + 8, pack_bf16(s[n] - bf16lo(w01), s[n + 1] - bf16hi(w01)), pack_bf16(s[n + 2] - bf16lo(w23), s[n + 3] - bf16hi(w23)));
              }
            }
          if (step == tail_step) clear_tail(step, tail);
          fence_proxy_async();
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
        }
        // a row's sum over the warp's lanes: half of the columns a step, until a lane has one
#pragma unroll
        for (int half = 0; half < 2; ++half)
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
                fap_tmem_ld(tO + g * OST + c0, o);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= f;
                tmem_st32(tO + g * OST + c0, reinterpret_cast<uint32_t*>(o));
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
          if (step == tail_step) clear_tail(step, tail);
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
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ------------------------------------------------------------------------------------------------ TMA
    if (warp == 8) {
      bool alive = true;
      int cq[2] = {0, 0}, ck = 0;   // pieces with a query tile g, key tiles, before this piece
      int turned = -RING - 1;       // the last key tile of the last piece of the turned kind
      // 8-bit pages: key tiles and pieces of the turned kind so far; of each place (those of V, then those of K) whether a tile of that kind, or another, was put there since it was last
      // waited for, and the parity of the wait.  (Each round of each barrier is waited for once, so that its parity tells it.)
      int cf = 0, few_pieces = 0;
      uint32_t few_in = 0, dense_in = 0, few_round = 0, dense_round = 0;
      auto acquire = [&](int place) {
        const uint32_t bit = 1u << place;
        if (few_in & bit) {
          if (!gemm_wait_warp(smem_u32(&f_empty[place]), (few_round >> place) & 1, abortp)) return false;
          few_in &= ~bit;
          few_round ^= bit;
        } else if (dense_in & bit) {
          if (!gemm_wait_warp(place < RING ? smem_u32(&v_empty[place]) : smem_u32(&k_empty[place - RING]), (dense_round >> place) & 1, abortp)) return false;
          dense_in &= ~bit;
          dense_round ^= bit;
        }
        return true;
      };
      for (int at = begin; alive && at < end; ++at) {
        if (at == begin + 1) asm volatile("bar.sync 5, 384;" ::: "memory");   // (the list is there)
        const int4* const e = at == begin ? reinterpret_cast<const int4*>(a.pieces + at) : chunk_words(a, list, begin, at);
        const int4 z = e[2];
        const int lead0 = z.y, lead1 = z.z;   // the pages of its first key tile
        ChunkPiece p;
        if (!chunk_read(a, e[0], e[1], z, p)) continue;
        // 8-bit pages: the last products of pieces of the turned kind before the last two are known here to be done, so that the two barriers tell the rounds apart.
        if (F8 && p.kind == CHUNK_FEW && few_pieces > 1 && !(alive = gemm_wait_warp(smem_u32(&turn_free[few_pieces & 1]), ((few_pieces >> 1) - 1) & 1, abortp))) break;
        const int32_t* const pages = a.table + (size_t)p.request * a.blocks;
        const int last_page = (p.pos0 + p.tokens - 1) / kStepPage;
        int first = 2 * p.k0, ids = __ldg(pages + min(first + lane, last_page));   // 32 pages from `first` on, a lane each; behind the last key: the last one
        auto fetch_q = [&](int g) {
          if ((p.kind == CHUNK_PAIR ? p.cnt(g) : F8 && p.kind == CHUNK_FEW ? 0 : 1 - g) == 0) return true;
          if (!gemm_wait_warp(smem_u32(&q_empty[g]), (cq[g] & 1) ^ 1, abortp)) return false;
          ++cq[g];
          // Q1 lies where P of the turned kind did: behind its last product, which frees the last tile of V (where that place was used since, it has)
          if constexpr (F8) {
            if (g && few_pieces > 0 && !gemm_wait_warp(smem_u32(&turn_free[(few_pieces - 1) & 1]), ((few_pieces - 1) >> 1) & 1, abortp)) return false;
          } else {
            if (g && ck - turned <= RING && !gemm_wait_warp(smem_u32(&v_empty[turned % RING]), (turned / RING) & 1, abortp)) return false;
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
        const bool codes = F8 && p.kind == CHUNK_FEW;
        for (int j = 0; j < p.n; ++j, codes ? ++cf : ++ck) {
          const int i = ck % RING, ph = (ck / RING) & 1;
          if (2 * (p.k0 + j) >= first + 32) {
            first += 32;
            ids = __ldg(pages + min(first + lane, last_page));
          }
          const int page0 = j == 0 ? lead0 : __shfl_sync(0xffffffffu, ids, 2 * (p.k0 + j) - first);
          const int page1 = j == 0 ? lead1 : __shfl_sync(0xffffffffu, ids, 2 * (p.k0 + j) + 1 - first);
          if constexpr (F8) {
            if (codes) {   // both pages of K, both of V, rows of D bytes in the swizzle of their length
              const int place = cf % T::PLACES;
              if (!(alive = acquire(place))) break;
              few_in |= 1u << place;
              if (lane == 0) {
                mbar_arrive_expect_tx(&f_full[place], T::TILE);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  fap_tma_4d(smV + place * T::TILE + r * (64 * D), r < 2 ? &codes8.k : &codes8.v, smem_u32(&f_full[place]), 0, 0, p.head, r & 1 ? page1 : page0);
              }
              continue;
            }
            if (!(alive = acquire(RING + i))) break;
            dense_in |= 1u << (RING + i);
          } else if (!(alive = gemm_wait_warp(smem_u32(&k_empty[i]), ph ^ 1, abortp))) break;
          fetch(&map_k, smK + i * T::TILE, &k_full[i], page0, page1);
          if (j == 0 && !(alive = fetch_q(1))) break;
          if constexpr (F8) {
            if (!(alive = acquire(i))) break;
            dense_in |= 1u << i;
          } else if (!(alive = gemm_wait_warp(smem_u32(&v_empty[i]), ph ^ 1, abortp))) break;
          fetch(&map_v, smV + i * T::TILE, &v_full[i], page0, page1);
        }
        if (p.kind == CHUNK_FEW) { turned = t0 + p.n - 1; ++few_pieces; }
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
      // scores of group g by query tile `tile`: S_g = Q K^T, or of the turned kind, whose rows' word of the instruction is `wide`, K Q^T
      auto qk = [&](int g, int tile, int t, uint32_t wide) {
        uint32_t dq = tile ? dq1 : dq0, dk = dk0 + (t % RING) * (T::TILE >> 4);
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
        uint32_t dv = dv0 + (t % RING) * (T::TILE >> 4);
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
      // 8-bit pages, turned kind: S^T = K Q^T, O^T += V^T P^T of the codes in a place; blocks: eights of rows
      auto qk8 = [&](int tile, int which, int blocks) {
        constexpr uint64_t UP = D == 128 ? UPPER : ((uint64_t)(512 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)4 << 61);   // (rows of 128 bytes, of 64)
        uint32_t dk = ((smV + tile % T::PLACES * T::TILE) & 0x3FFFF) >> 4, dq = ((smF + which * T::QF) & 0x3FFFF) >> 4;
        asm volatile("" : "+r"(dq), "+r"(dk));
        const uint32_t id = (1u << 4) | ((uint32_t)(2 * blocks) << 17) | ((128u >> 4) << 24);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) chunk_mma_f8(tm + COL_S + (tile & 1) * 128 + 32 * (tile & 2), UP | (dk + 2 * k), UP | (dq + 2 * k), id, k > 0 ? 1u : 0u);
        fap_commit(&fs_full[tile & 3]);
      };
      auto pv8 = [&](int tile, bool first, int blocks) {
        // V with its rows (keys) for K: eight of them D bytes each an atom; behind the first D features of 128 rows of A there are none at head size 64 (what lies 8 KB on)
        constexpr uint64_t UP = ((uint64_t)(8 * D >> 4) << 32) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)1 << 46) | ((uint64_t)(D == 128 ? 2 : 4) << 61);
        uint32_t dv = ((smV + tile % T::PLACES * T::TILE + 128 * D) & 0x3FFFF) >> 4, dp = dq1 + (tile & 1) * (T::P >> 4);
        asm volatile("" : "+r"(dv), "+r"(dp));
        const uint32_t id = (1u << 4) | (1u << 10) | (1u << 15) | ((uint32_t)((3 * blocks + 1) / 2 * 2) << 17) | ((128u >> 4) << 24);
#pragma unroll
        for (int k = 0; k < 4; ++k) chunk_mma_f8(tm + COL_O + (tile & 1) * OST, UP | (dv + k * (32 * D >> 4)), UPPER | (dp + 2 * k), id, (!first || k > 0) ? 1u : 0u);
        fap_commit(&fo_full[tile & 1]);
        fap_commit(&f_empty[tile % T::PLACES]);
      };
      auto wide_of = [&](const ChunkPiece& p) { return p.kind == CHUNK_FEW ? (uint32_t)((p.tokens * a.G + 15) / 16 * 2) << 17 : 0u; };
      int cf = 0, few_pieces = 0, scored = 0;      // 8-bit pages: key tiles and pieces of the turned kind before this piece, which ck leaves out; tiles whose scores were asked for
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
      auto wait_k = [&](int t) { alive &= gemm_wait(smem_u32(&k_full[t % RING]), (t / RING) & 1, abortp); };
      auto wait_v = [&](int t) { alive &= gemm_wait(smem_u32(&v_full[t % RING]), (t / RING) & 1, abortp); };
      // the first scores of group g of piece p, whose key tiles begin at tile t and whose query tiles are number q0, q1
      auto open = [&](const ChunkPiece& p, int g, int t, int q0, int q1) {
        const bool pair = p.kind == CHUNK_PAIR;
        const int tile = pair ? g : 0, step = pair ? 0 : g;
        alive &= gemm_wait(smem_u32(&q_full[tile]), (tile ? q1 : q0) & 1, abortp);
        wait_k(t + step);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (elect_one() && alive) {
          qk(g, tile, t + step, wide_of(p));
          if (!pair) fap_commit(&k_empty[(t + step) % RING]);                    // (of a pair, both tiles read the same keys)
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
        const bool pair = p.kind == CHUNK_PAIR;
        if constexpr (F8) {
          if (p.kind == CHUNK_FEW) {
            // Scores as soon as their tile is there and one of the four places for them is free (which the weights of the tile four before say), products as soon as their weights are.
            const int end_own = cf + p.n, end_all = more && next.kind == CHUNK_FEW ? end_own + next.n : end_own;
            int tile = cf, idle = 0;
            alive = __all_sync(0xffffffffu, alive);
            while (alive && tile < end_own) {
              bool moved = false;
              if (scored < min(tile + 4, end_all)) {
                const bool own = scored < end_own;
                const int which = (few_pieces + !own) & 1, place = scored % T::PLACES;
                if (chunk_ready(&qf_full[which], ((few_pieces + !own) >> 1) & 1) && chunk_ready(&f_full[place], (scored / T::PLACES) & 1)) {
                  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                  if (elect_one()) {
                    qk8(scored, which, ((own ? p.tokens : next.tokens) * a.G + 7) / 8);
                    if (scored + 1 == (own ? end_own : end_all)) fap_commit(&qf_empty[which]);
                  }
                  ++scored;
                  moved = true;
                }
              }
              if (tile < scored && chunk_ready(&fp_full[tile & 1], (tile >> 1) & 1)) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                  pv8(tile, tile < cf + 2, (p.tokens * a.G + 7) / 8);
                  if (tile + 1 == end_own) fap_commit(&turn_free[few_pieces & 1]);
                }
                ++tile;
                moved = true;
              }
              idle = moved ? 0 : idle + 1;
              if (__any_sync(0xffffffffu, idle > (int)kGemmWaitLimit || *abortp)) {
                *abortp = 1;
                if (lane == 0) atomicExch(&g_gemm_error, 1u);
                alive = false;
              }
            }
            if (!alive) break;
            cf = end_own; ++few_pieces;
            continue;
          }
        }
        const int tn = ck + p.n;                   // the next piece's first key tile
        const int nq0 = cq[0] + (pair ? p.cnt0 > 0 : 1), nq1 = cq[1] + (pair && p.cnt1 > 0);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (p.cnt(g) > 0 && !ahead[g]) open(p, g, ck, cq[0], cq[1]);
          ahead[g] = false;
        }
        // the next piece's scores, while this one's last tiles and its O are worked on
        // (The second key tile's scores come behind the first's: the last ones give Q's place up.  8-bit pages: a piece of the turned kind uses the places that this one holds.)
        auto go_on = [&](int g) {
          if (more && !(F8 && next.kind == CHUNK_FEW) && next.cnt(g) > 0 && (next.kind == CHUNK_PAIR || g == 0 || ahead[0])) {
            open(next, g, tn, nq0, nq1);
            ahead[g] = true;
          }
        };
        if (pair) {
          if (elect_one() && alive) fap_commit(&k_empty[ck % RING]);
          for (int j = 0; j < p.n; ++j) {
            const int t = ck + j;
            wait_v(t);
            if (j + 1 < p.n) wait_k(t + 1);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int ng = p.cnt(g);
              if (j < ng) {
                alive &= gemm_wait(smem_u32(&p_full[g]), (c[g] + j) & 1, abortp);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one() && alive) {
                  pv(g, t, j == 0, 0);
                  if (j + 1 < ng) {
                    qk(g, g, t + 1, 0);
                    if (j + 2 == ng) fap_commit(&q_empty[g]);
                  }
                }
                // (the turned kind's P goes where Q1 is: not before this piece's last scores of tile 1 are on their way)
                if (j + 1 == ng && (next.kind != CHUNK_FEW || g || j + 1 == p.n)) go_on(g);
              }
            }
            if (elect_one() && alive) {
              fap_commit(&v_empty[t % RING]);
              if (j + 1 < p.n) fap_commit(&k_empty[(t + 1) % RING]);
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
              fap_commit(&v_empty[t % RING]);
            }
            if (j + 2 < p.n) {
              wait_k(t + 2);
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              if (elect_one() && alive) {
                qk(g, 0, t + 2, wide);
                fap_commit(&k_empty[(t + 2) % RING]);
                if (j + 3 == p.n) fap_commit(&q_empty[0]);
              }
            } else if (!(wide && next.kind == CHUNK_PAIR && g && j + 1 < p.n)) {   // (Q1 of a pair comes behind the last product that reads P)
              go_on(g);
            }
          }
        }
        c[0] += p.cnt0; c[1] += p.cnt1; ck = tn;
        cq[0] = nq0; cq[1] = nq1;
      }
    }
    // ------------------------------------------------------------------------------------------------ scales of 8-bit pages
    if (F8 && warp == 10) {
      bool alive = true;
      int cf = 0;
      int at = begin;
      ChunkPiece p;
      while (alive && chunk_piece(a, list, begin, at, end, p)) {
        if (p.kind != CHUNK_FEW) continue;
        const int32_t* const pages = a.table + (size_t)p.request * a.blocks;
        const int last_page = (p.pos0 + p.tokens - 1) / kStepPage;
        int first = 2 * p.k0;
        float to_log2, value;   // of 32 pages from `first` on, a lane each
        auto read = [&]() {
          const size_t e = (size_t)__ldg(pages + min(first + lane, last_page)) * a.Hkv + p.head;
          to_log2 = __ldg(a.k_scales + e) * a.scale_log2e;
          value = __ldg(a.v_scales + e);
          value = value < 0x1p-60f ? 0x1p-60f : value;   // (0, as pools begin, with codes of 0)
        };
        read();
        for (int j = 0; j < p.n; ++j, ++cf) {
          if (2 * (p.k0 + j) >= first + 32) {
            first += 32;
            read();
          }
          const int i = cf % kChunkScales, at0 = 2 * (p.k0 + j) - first;
          if (!(alive = gemm_wait_warp(smem_u32(&sc_empty[i]), ((cf / kChunkScales) & 1) ^ 1, abortp))) break;
          if (lane == at0 || lane == at0 + 1) sc[i][lane - at0] = make_float4(to_log2, log2f(value), 1.f / value, 0.f);
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&sc_full[i]);
          }
        }
      }
    }
    // ------------------------------------------------------------------------------------------------ queries of few rows as codes
    if (F8 && warp == 11) {
      bool alive = true;
      int at = begin, n = 0;
      ChunkPiece p;
      while (alive && chunk_piece(a, list, begin, at, end, p)) {
        if (p.kind != CHUNK_FEW) continue;
        const int rows = p.tokens * a.G, which = n & 1;
        const uint32_t smq = smF + which * T::QF;
        bool waited = n < 2;   // (rows come from memory meanwhile)
        // D / 16 lanes a row, 16 features each
        for (int x = lane; x < (rows + 7) / 8 * 8 * (D / 16); x += 32) {
          const int row = x / (D / 16), c16 = x % (D / 16), tok = row / a.G;
          uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
          if (row < rows) {
            const uint4* const from = reinterpret_cast<const uint4*>(a.q + (p.row0 + tok) * a.q_row + (p.head * a.G + row - tok * a.G) * a.q_head) + 2 * c16;
            v[0] = __ldg(from);
            v[1] = __ldg(from + 1);
          }
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            constexpr uint32_t ABS = 0x7fff7fffu;
            m = __vmaxu2(__vmaxu2(__vmaxu2(m, v[i].x & ABS), __vmaxu2(v[i].y & ABS, v[i].z & ABS)), v[i].w & ABS);
          }
          m = max(m & 0xffffu, m >> 16);
#pragma unroll
          for (int k = 1; k < D / 16; k <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, k));   // (whole warps come here: eight rows are 64 or 32 pieces)
          if (!waited) {
            waited = true;
            if (!(alive = gemm_wait_warp(smem_u32(&qf_empty[which]), ((n >> 1) - 1) & 1, abortp))) break;
          }
          // The largest becomes 2^7 and a little (rows of less than 2^-95, whose scores are 0, as they are; an infinity or a NaN makes the row's scores NaN).
          const int e = m < 0x1000u ? 127 + 7 : min((int)(m >> 7), 254);
          const float up = __uint_as_float((uint32_t)(127 + 7 + 127 - e) << 23);
          if (c16 == 0) q_scale[which][row] = m >= 0x7f80u ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)(e - 7) << 23);
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4& u = v[i >> 1];
            const uint32_t w0 = i & 1 ? u.z : u.x, w1 = i & 1 ? u.w : u.y;
            const float v0 = bf16lo(w0) * up, v1 = bf16hi(w0) * up, v2 = bf16lo(w1) * up, v3 = bf16hi(w1) * up;
            float c0, c1, c2, c3;
            hi[i] = chunk_codes4(v0, v1, v2, v3);
            chunk_f32(chunk_f16(hi[i]), c0, c1);
            chunk_f32(chunk_f16(hi[i] >> 16), c2, c3);
            lo[i] = chunk_codes4(v0 - c0, v1 - c1, v2 - c2, v3 - c3);
          }
          const uint32_t to = smq + (row >> 3) * (16 * D) + chunk_code_at<D>(row & 7, c16);   // eight rows' first numbers, their second ones, ...
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to + 8 * D), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
        }
        if (!alive) break;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&qf_full[which]);
        ++n;
      }
    }
    // ------------------------------------------------------------------------------------------------ rows behind the last request's
    if (warp == (F8 ? 11 : 10) && a.rest) {
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

template <int D, bool F8, class Codes>
static cudaError_t launch_chunk(const CUtensorMap (&m)[4], const Codes& codes, const ChunkArgs& a, cudaStream_t st) {
  using T = ChunkTile<D, F8>;
  static std::atomic<unsigned long long> served{0};
  const cudaError_t set = once_per_device(served, [] {
    cudaFuncAttributes at;
    const cudaError_t e = cudaFuncGetAttributes(&at, chunk_attn_kernel<D, F8>);
    if (e != cudaSuccess) return e;
    // the warps' register shares must fit what the block is launched with, or they would wait for registers for good
    if (at.numRegs * T::THREADS < 8 * 32 * 216 + 4 * 32 * 64) return cudaErrorInvalidConfiguration;
    return cudaFuncSetAttribute(chunk_attn_kernel<D, F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
  });
  if (set != cudaSuccess) return set;
  count_launch();
  return launch_pdl(chunk_attn_kernel<D, F8>, dim3((unsigned)(num_sms() < kStepMaxCtas ? num_sms() : kStepMaxCtas)), dim3(T::THREADS), T::SMEM, st, m[0], m[1], m[2], m[3], codes, a);
}

// 8-bit pages of the requests that have more rows than the turned kind takes, as bf16 where they will be read as those are: the tensor cores' operands of that kind come from shared memory
// alone, and every query tile would turn the same codes around again.  (Four warps beside the softmax's that widened them tile by tile: 2048 tokens behind 15000 812 us and more; so 502; pages of 16 bits 469.)  A block (page, head) a CTA at a time.
__global__ void __launch_bounds__(256) chunk_widen_kernel(const uint8_t* k8, const uint8_t* v8, const float* ks, const float* vs, uint16_t* k16, uint16_t* v16, const int32_t* row_starts,
                                                          const int32_t* contexts, const int32_t* table, int requests, int blocks, int Hkv, int D, int few_tokens) {
  __shared__ int list[256];   // requests of this round that have so many
  __shared__ int of_warp[8];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, pieces = 64 * D / 16;   // of 16 codes, of a block of K or of V
  int done = 0;                                        // blocks before this request's, so that the CTAs have equal shares of all
  for (int s0 = 0; s0 < requests; s0 += 256) {
    const int s = s0 + tid;
    const bool many = s < requests && __ldg(row_starts + s + 1) - __ldg(row_starts + s) > few_tokens;
    const unsigned who = __ballot_sync(0xffffffffu, many);
    if ((tid & 31) == 0) of_warp[tid >> 5] = __popc(who);
    __syncthreads();
    int n = 0, before = __popc(who & ((1u << (tid & 31)) - 1));
    for (int w = 0; w < 8; ++w) {
      if (w == tid >> 5) before += n;
      n += of_warp[w];
    }
    if (many) list[before] = s;
    __syncthreads();
    for (int i = 0; i < n; ++i) {
      const int r = list[i], keys = __ldg(contexts + r) + __ldg(row_starts + r + 1) - __ldg(row_starts + r), units = (keys + kStepPage - 1) / kStepPage * Hkv;
      for (int u = ((int)blockIdx.x + (int)gridDim.x - done % (int)gridDim.x) % (int)gridDim.x; u < units; u += gridDim.x) {
        const size_t block = (size_t)__ldg(table + (size_t)r * blocks + u / Hkv) * Hkv + u % Hkv;
        const float fk = __ldg(ks + block), fv = __ldg(vs + block);
        uint4 w[4];   // all of a thread's on their way together: at most two of K, two of V
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int e = tid + 256 * (q & 1);
          if (e < pieces) w[q] = __ldg(reinterpret_cast<const uint4*>(q >> 1 ? v8 : k8) + block * pieces + e);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int e = tid + 256 * (q & 1);
          if (e >= pieces) continue;
          const float f = q >> 1 ? fv : fk;
          const uint32_t in[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
          uint32_t out[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float lo, hi;
            chunk_f32(chunk_f16(in[i >> 1] >> (16 * (i & 1))), lo, hi);
            out[i] = pack_bf16(lo * f, hi * f);   // (exact: the scale is a power of two)
          }
          uint4* const to = reinterpret_cast<uint4*>(q >> 1 ? v16 : k16) + 2 * (block * pieces + e);
          to[0] = make_uint4(out[0], out[1], out[2], out[3]);
          to[1] = make_uint4(out[4], out[5], out[6], out[7]);
        }
      }
      done += units % (int)gridDim.x;
    }
    __syncthreads();
  }
}
// whether some request may have more rows than the turned kind takes
static bool chunk_wide8(const pie_step_dims& d) { return d.rows > ChunkTile<128, true>::FEW / (d.Hq / d.Hkv); }
static cudaError_t launch_chunk_widen(const ChunkArgs& a, const pie_step_dims& d, int D, const uint8_t* k8, const uint8_t* v8, uint16_t* k16, uint16_t* v16, cudaStream_t st) {
  count_launch();
  return launch_pdl(chunk_widen_kernel, dim3((unsigned)(num_sms() * 8)), dim3(256), 0, st, k8, v8, a.k_scales, a.v_scales, k16, v16, a.row_starts, a.contexts, a.table, d.requests, d.blocks,
                    d.Hkv, D, a.few_tokens);
}
static size_t chunk_workspace_bytes(int D) { return kStepMaxCtas * 4 + (size_t)2 * kStepMaxCtas * (D == 128 ? kChunkRecord<128> : kChunkRecord<64>) * 4; }
// the common part: q's maps, the plan's arrays
template <bool F8>
static int chunk_common(ChunkArgs& a, CUtensorMap* maps, void* out, const pie_head_rows* q, const void* kpool, const void* vpool, const int32_t* plan, const pie_step_dims* d, int D, float scale, int rest,
                        void* workspace, size_t workspace_bytes) {
  if ((D != 64 && D != 128) || !(scale > 0.f) || scale > 3.4028234e38f / 1.5f || q->stride_h % 8 || q->stride_l % 8 || (d->rows > 1 && q->stride_l <= 0) ||
      (d->Hq > 1 && q->stride_h <= 0))
    return PIE_EINVAL_SHAPE;
  for (const void* p : {(const void*)out, q->p, kpool, vpool, (const void*)plan, (const void*)workspace})
    if (reinterpret_cast<uintptr_t>(p) & 15) return PIE_EALIGN;
  if (!workspace || workspace_bytes < chunk_workspace_bytes(D)) return PIE_EWORKSPACE;
  const StepLayout l = step_layout(*d);
  a = {};
  a.out = (uint16_t*)out; a.Hq = d->Hq; a.Hkv = d->Hkv; a.G = d->Hq / d->Hkv; a.tile_tokens = l.tile_tokens; a.rows = d->rows; a.requests = d->requests;
  a.scale_log2e = scale * 1.4426950408889634f;
  a.ranges = plan + l.ranges; a.table = plan + l.block_table; a.row_starts = plan + l.row_starts; a.contexts = plan + l.contexts;
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
  if (int s = chunk_common<false>(a, maps, out, q, kpool, vpool, plan, d, D, scale, rest, workspace, workspace_bytes)) return s;
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
  return status_of(D == 128 ? launch_chunk<128, false>(maps, ChunkNone{}, a, (cudaStream_t)stream) : launch_chunk<64, false>(maps, ChunkNone{}, a, (cudaStream_t)stream));
}

// the workspace: that of pie_chunk_attn, and room for a layer's pools in 16 bits where a request may have more rows than the turned kind takes
size_t pie_chunk_attn_fp8_workspace_bytes(const pie_step_dims* d, int D) {
  if (step_dims_status(d) || (D != 64 && D != 128)) return 0;
  return chunk_workspace_bytes(D) + (chunk_wide8(*d) ? (size_t)d->pages * d->Hkv * kStepPage * D * 4 : 0);
}

int pie_chunk_attn_fp8(void* out, const pie_head_rows* q, const uint8_t* kpool, const float* k_scales, const uint8_t* vpool, const float* v_scales, const int32_t* plan,
                       const pie_step_dims* d, int D, float scale, int rest, void* workspace, size_t workspace_bytes, void* stream) {
  if (int s = step_dims_status(d)) return s;
  if (!out || !q || !q->p || !kpool || !k_scales || !vpool || !v_scales || !plan) return PIE_ENULL;
  ChunkArgs a;
  CUtensorMap maps[4];
  if (D == 64 || D == 128)
    if (!workspace || workspace_bytes < pie_chunk_attn_fp8_workspace_bytes(d, D)) return PIE_EWORKSPACE;
  if (int s = chunk_common<true>(a, maps, out, q, kpool, vpool, plan, d, D, scale, rest, workspace, workspace_bytes)) return s;
  a.k_scales = k_scales; a.v_scales = v_scales;
  a.q = (const uint16_t*)q->p; a.q_row = d->rows > 1 ? q->stride_l : 0; a.q_head = d->Hq > 1 ? q->stride_h : 0;
  const GemmEncodeFn fn = gemm_encode_fn();
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const bool wide = chunk_wide8(*d);
  const cuuint64_t block = (cuuint64_t)kStepPage * D, dims[4] = {(cuuint64_t)D, (cuuint64_t)kStepPage, (cuuint64_t)d->Hkv, (cuuint64_t)d->pages};
  const size_t half = (size_t)d->pages * d->Hkv * kStepPage * D;
  uint16_t* const k16 = (uint16_t*)((uint8_t*)workspace + chunk_workspace_bytes(D));
  ChunkMaps8 codes;
  for (int i = 0; i < 2; ++i) {   // a page of one head: 64 rows of D bytes; and in 16 bits, 64 features of them
    const cuuint64_t strides[3] = {(cuuint64_t)D, block, block * d->Hkv}, strides16[3] = {2 * (cuuint64_t)D, 2 * block, 2 * block * d->Hkv};
    const cuuint32_t box[4] = {(cuuint32_t)D, (cuuint32_t)kStepPage, 1, 1}, box16[4] = {64, 64, 1, 1};
    if (fn(i ? &codes.v : &codes.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(i ? vpool : kpool), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return PIE_EUNSUPPORTED;
    maps[2 + i] = maps[0];        // (no piece asks for it)
    if (wide && fn(&maps[2 + i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, i ? k16 + half : k16, dims, strides16, box16, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return PIE_EUNSUPPORTED;
  }
  const cudaStream_t st = (cudaStream_t)stream;
  if (wide)
    if (const cudaError_t e = launch_chunk_widen(a, *d, D, kpool, vpool, k16, k16 + half, st); e != cudaSuccess) return status_of(e);
  return status_of(D == 128 ? launch_chunk<128, true>(maps, codes, a, st) : launch_chunk<64, true>(maps, codes, a, st));
}

}  // extern "C"
