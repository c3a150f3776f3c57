// A ragged step -- every request brings another number of new tokens -- described on the device (BatchDetails, CORE/include/engine/batch_details.hpp:10-90, is
// the host's form of it), and the rotation and cache write of its rows.
#include "pie_ptx.cuh"
#include "pie_step_plan.h"

namespace pie {

int step_dims_status(const pie_step_dims* d) {
  if (!d) return PIE_ENULL;
  if (d->requests < 1 || d->requests > kStepMaxRequests || d->rows < 1 || d->logit_rows < 1 || d->blocks < 1 || d->pages < 1 || d->Hq < 1 || d->Hkv < 1 ||
      d->Hq % d->Hkv || d->Hq / d->Hkv > kStepTile || (long long)d->requests * d->blocks > 0x7fffffff || (long long)d->pages * kStepPage > 0x7fffffff ||
      (long long)d->blocks * kStepPage > 0x7fffffff - kStepRoom || (long long)d->rows * d->Hq > 0x7fffffff || step_layout(*d).items > 0x3fffffff)
    return PIE_EINVAL_SHAPE;
  return PIE_OK;
}

// ---------------------------------------------------------------------------------------------------- the plan
// Every array of the plan is a function of four sums over the requests before one (rows, pages, logit rows, cost of attention).  One launch: each CTA takes the sums of
// all requests itself, in shared memory (at most 4096 of them), and fills its part of every array, finding a row's request by bisection.  Kilobytes: what counts is one
// launch and the length of the chain load, scan, bisection, page id, store.  8 requests 6.0 us, 212 requests of 11700 rows 7.0, in a row of such launches; a call costs its
// host 8.
//
// Attention's work is dealt out to the SMs in equal shares: items (key / value head, request, pair of query tiles) lie on a line, as long as they have keys to multiply
// (twice that where both query tiles have rows) and a constant for what an item costs besides; CTA c has [c share, (c + 1) share) of the line.  An item that lies in
// several shares is cut between key tiles, and its pieces are added up by the last CTA to finish one (pie_chunk_attn.cuh).  A CTA has pieces of at most two cut items, so
// the space for partial results is known.  Which keys are added up where depends on the lengths alone.
struct PlanArgs {
  int32_t* plan;
  pie_step_dims d;
  StepLayout l;
  const int32_t *ids, *input, *context, *draft, *pages;
  long long n_page_ids, page_stride;
  int ctas;
};
constexpr int kPlanThreads = 512;
constexpr int kCostPair = 2, kCostTile = 1;   // a key of an item with rows in both query tiles, in one (powers of two)
// Queries in, results out.  Over 27 steps of both head sizes, 1 to 212 requests, answers, drafts and portions, a flat choice: 256 and 960 stay within 5 % of it either way but for one answer of
// 9000 keys (256: 28.6 us, this 26.2), a prompt of 8192 (528, 500), 4 answers with drafts over 1000 (21.0, 19.6; 960: 17.9) and 16 with up to 14 drafts over 4000 (960: 84.8, 79.0).
constexpr int kCostItem = 576;
static_assert(kCostItem < kStepRoom && kStepTile < kStepRoom, "added to keys in 32 bits");
constexpr long long kCostShare = 512;         // least share worth a CTA; without pairs of query tiles, whose keys are sooner read than added up in pieces, twice that
static_assert(kCostTile * kStepTile == 1 << 7 && kCostPair * kStepTile == 1 << 8, "key tiles are counted by shifts");
constexpr int kCutPair = 4, kCutTile = 2;     // least key tiles of a piece: what it costs to leave a piece's results and to add them up

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
// exclusive sums over the block's threads, N at a time
template <int N>
__device__ __forceinline__ void block_scan(long long (&v)[N], long long* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kPlanThreads / 32;
  long long inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    inc[i] = warp_scan(v[i], lane);
    if (lane == 31) sm[i * warps + warp] = inc[i];
  }
  __syncthreads();
  if (warp < N) {
    const long long t = warp_scan(lane < warps ? sm[warp * warps + lane] : 0, lane);
    if (lane < warps) sm[warp * warps + lane] = t;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = inc[i] - v[i] + (warp ? sm[i * warps + warp - 1] : 0);
  __syncthreads();
}
// the last index i < n with first[i] <= x of a rising sequence that begins at or below x: of equal ones the last
template <class T>
__device__ __forceinline__ int last_at_or_below(const T* first, int n, T x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// cost of the first q items of a request, all of them full
__device__ __forceinline__ long long cost_before(long long q, int context, int span) {
  return q * ((long long)kCostPair * context + kCostItem) + (long long)kCostPair * span * (q * (q + 1) / 2);
}

__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ __align__(16) uint8_t plan_smem[];
  __shared__ long long scan_sm[3 * (kPlanThreads / 32)];
  __shared__ long long page_total, row_total;
  __shared__ int bad, kinds;
  const int S = a.d.requests, T = a.d.rows, tid = threadIdx.x, span = 2 * a.l.tile_tokens;
  long long* const cost = reinterpret_cast<long long*>(plan_smem);   // [S + 1] each
  int* const row = reinterpret_cast<int*>(cost + S + 1);
  int* const page = row + S + 1;
  int* const logit = page + S + 1;
  int* const item = logit + S + 1;
  int* const ctx = item + S + 1;
  pdl_launch_dependents();
  pdl_wait();
  if (tid == 0) bad = kinds = 0;
  __syncthreads();
  int fault = 0;

  // ---- the sums: each thread a run of requests
  const int per = (S + kPlanThreads - 1) / kPlanThreads, s0 = min(tid * per, S), s1 = min(s0 + per, S);
  auto lengths = [&](int s, int& n, int& c) {   // checked; 0, 0 where they cannot be
    n = __ldg(a.input + s);
    c = __ldg(a.context + s);
    if (n < 0 || c < 0 || n > T || (long long)n + c > (long long)a.d.blocks * kStepPage) {
      n = c = 0;
      return false;
    }
    return true;
  };
  {
    long long v[2] = {0, 0};
    for (int s = s0; s < s1; ++s) {
      int n, c;
      if (!lengths(s, n, c)) fault |= PIE_STEP_LENGTH;
      v[0] += n;
      v[1] += (n + c + kStepPage - 1) / kStepPage;
    }
    block_scan(v, scan_sm);
    for (int s = s0; s < s1; ++s) {
      int n, c;
      lengths(s, n, c);
      row[s] = (int)min(v[0], (long long)T);
      page[s] = (int)min(v[1], 0x7fffffffLL);
      ctx[s] = c;
      v[0] += n;
      v[1] += (n + c + kStepPage - 1) / kStepPage;
      if (v[0] > T) fault |= PIE_STEP_ROWS;
    }
    if (s0 < S && s1 == S) { row[S] = (int)min(v[0], (long long)T); page[S] = (int)min(v[1], 0x7fffffffLL); row_total = v[0]; page_total = v[1]; }
  }
  __syncthreads();
  if (!a.page_stride && page_total > a.n_page_ids) fault |= PIE_STEP_PAGES;
  {
    long long v[3] = {0, 0, 0};
    auto add = [&](int s, long long (&v)[3]) {
      const int n = row[s + 1] - row[s];
      if (n == 0) return;
      int dr = a.draft ? __ldg(a.draft + s) : 0;
      int all = n;
      if (row_total > T) {   // rows that are cut off take their drafts with them
        int c;
        lengths(s, all, c);
      }
      if (dr < 0 || dr >= all) { fault |= PIE_STEP_DRAFT; dr = 0; }
      dr = max(0, dr - (all - n));
      const int full = (n - 1) / span, rest = n - full * span;
      v[0] += dr + 1;
      v[1] += full + 1;
      v[2] += cost_before(full, ctx[s], span) + (long long)(rest > a.l.tile_tokens ? kCostPair : kCostTile) * (ctx[s] + n) + kCostItem;
    };
    for (int s = s0; s < s1; ++s) add(s, v);
    block_scan(v, scan_sm);
    int kind = 0;   // 1: a pair of query tiles, 2: an item of more than the larger least share (where there is none, a CTA an item)
    for (int s = s0; s < s1; ++s) {
      const int n = row[s + 1] - row[s];
      kind |= (n > a.l.tile_tokens ? 1 : 0) | (n > 0 && ctx[s] + n + kCostItem > 2 * kCostShare ? 2 : 0);
      logit[s] = (int)v[0];   // (at most T; what lies behind the last logit row is cut off below)
      item[s] = (int)v[1];
      cost[s] = v[2];
      add(s, v);
      if (v[0] > a.d.logit_rows) fault |= PIE_STEP_LOGITS;
    }
    if (kind) atomicOr(&kinds, kind);
    if (s0 < S && s1 == S) { logit[S] = (int)v[0]; item[S] = (int)v[1]; cost[S] = v[2]; }
  }
  __syncthreads();

  // ---- the arrays
  const int first = blockIdx.x * kPlanThreads + tid, step = gridDim.x * kPlanThreads;
  int32_t* const w = a.plan;
  // a request's page, or -1
  auto page_id = [&](int s, int j) {
    int id = -1;
    if (a.page_stride) {
      if (j < a.n_page_ids) id = __ldg(a.pages + s * a.page_stride + j);
      else fault |= PIE_STEP_PAGES;
    } else {
      const long long at = (long long)page[s] + j;
      if (at < a.n_page_ids) id = __ldg(a.pages + at);
      else return -1;
    }
    if (id < 0 || id >= a.d.pages) { fault |= PIE_STEP_PAGE_ID; id = -1; }
    return id;
  };
  for (int s = first; s <= S; s += step) {
    w[a.l.row_starts + s] = row[s];
    w[a.l.logit_starts + s] = min(logit[s], a.d.logit_rows);
    if (s < S) w[a.l.contexts + s] = ctx[s];
  }
  auto do_row = [&](int t) {
    int s = -1, p = 0, slot = -1;
    if (t < row[S]) {
      s = last_at_or_below(row, S, t);
      p = ctx[s] + t - row[s];
      const int id = page_id(s, p / kStepPage);
      if (id >= 0) slot = id * kStepPage + p % kStepPage;
    }
    w[a.l.sequences + t] = s;
    w[a.l.positions + t] = p;
    w[a.l.slots + t] = slot;
  };
  const unsigned cells = (unsigned)S * (unsigned)a.d.blocks;
  auto do_cell = [&](unsigned e) {
    const int s = e / (unsigned)a.d.blocks, j = e % (unsigned)a.d.blocks;
    w[a.l.block_table + e] = j < page[s + 1] - page[s] ? max(page_id(s, j), 0) : 0;
  };
  auto do_logit = [&](int r) {
    int of = 0, token = -1;
    if (r < logit[S]) {
      const int s = last_at_or_below(logit, S, r), left = logit[s + 1] - 1 - r;
      of = row[s + 1] - 1 - left;
      if (left > 0 && r + 1 < a.d.logit_rows) token = __ldg(a.ids + of + 1);   // (a row that is the last one because of the cut judges none)
    }
    w[a.l.logit_rows + r] = of;
    w[a.l.draft_tokens + r] = token;
  };

  // ---- attention's schedule
  const int Q = item[S];
  const long long W1 = cost[S], W = W1 * a.d.Hkv;
  const long long least = kinds == 2 ? 2 * kCostShare : kCostShare;
  const long long want = max(1LL, min((long long)a.ctas, W / least)), share = (W + want - 1) / want;
  int32_t* const ranges = w + a.l.ranges;
  if (blockIdx.x == 0)
    for (int c = tid; c < kStepMaxCtas; c += kPlanThreads)
      if (c * share >= W) ranges[2 * c] = ranges[2 * c + 1] = 0;   // (the shares before it are written below)
  StepPiece* const pieces = reinterpret_cast<StepPiece*>(w + a.l.pieces);
  auto share_of = [&](long long at) { return W <= 0xffffffffLL ? (int)((uint32_t)at / (uint32_t)share) : (int)(at / share); };
  auto do_item = [&](int i) {
    const int head = i / Q, at = i - head * Q, s = last_at_or_below(item, S, at), q = at - item[s];
    const int n = row[s + 1] - row[s], tokens = min(span, n - q * span), keys = ctx[s] + q * span + tokens;
    const int weight = tokens > a.l.tile_tokens ? kCostPair : kCostTile, tiles = (keys + kStepTile - 1) / kStepTile;
    const long long x = head * W1 + cost[s] + cost_before(q, ctx[s], span), end = x + (long long)weight * keys + kCostItem;
    const int cut = weight == kCostPair ? kCutPair : kCutTile;
    auto tile = [&](int c) {   // first key tile of CTA c's share.  A cut that would leave little on one side of it is not made.
      const long long past = c * share - x;
      if (past <= 0) return 0;
      const int log = weight == kCostPair ? 8 : 7;   // of the cost of a key tile
      const long long k = (past + (1 << log) - 1) >> log;
      if (k < cut) return 2 * k <= tiles || tiles >= 2 * cut ? 0 : tiles;
      return tiles - k < cut ? tiles : (int)k;
    };
    const int c0 = share_of(x), c1 = share_of(end - 1);
    int mine = 0, opens = c0;
    for (int c = c0; c <= c1; ++c)
      if (tile(c) < tile(c + 1)) {
        if (mine == 0) opens = c;
        ++mine;
      }
    for (int c = c0; c <= c1; ++c) {
      StepPiece p;
      p.row0 = row[s] + q * span; p.pos0 = ctx[s] + q * span; p.tokens = tokens;
      p.request = s; p.kv_head = head;
      p.k0 = tile(c); p.k1 = tile(c + 1);
      p.first_cta = opens; p.pieces = mine;
      const int last_page = (keys - 1) / kStepPage;   // (behind the last key: its page again)
      for (int h = 0; h < 2; ++h) p.pages[h] = p.k0 < p.k1 ? max(page_id(s, min(2 * p.k0 + h, last_page)), 0) : 0;
      p.pad = 0;
      const int4* const from = reinterpret_cast<const int4*>(&p);
      int4* const to = reinterpret_cast<int4*>(pieces + i + c);   // the CTAs' lists lie one behind the other, with holes where an item ends with a share
      to[0] = from[0]; to[1] = from[1]; to[2] = from[2];
      if (c * share >= x) {   // the CTA's share begins in this item, and the one before it ends there or with the item before
        ranges[2 * c] = i + c;
        if (c > 0) ranges[2 * c - 1] = i + c - (c * share == x ? 1 : 0);
      }
    }
    if (i == Q * a.d.Hkv - 1) ranges[2 * c1 + 1] = i + c1 + 1;
  };

  // ---- one entry a thread: the arrays lie behind one another here, so that no thread waits for memory once for each
  const long long e0 = (long long)Q * a.d.Hkv, e1 = e0 + cells, e2 = e1 + T, e3 = e2 + a.d.logit_rows;
  for (long long e = first; e < e3; e += step) {
    if (e < e0) do_item((int)e);
    else if (e < e1) do_cell((unsigned)(e - e0));
    else if (e < e2) do_row((int)(e - e1));
    else do_logit((int)(e - e2));
  }

  if (fault) atomicOr(&bad, fault);
  __syncthreads();
  if (tid == 0) w[a.l.status + blockIdx.x] = bad;
  if (blockIdx.x == 0)
    for (int c = (int)gridDim.x + tid; c < kStepMaxCtas; c += kPlanThreads) w[a.l.status + c] = 0;
}

// ---------------------------------------------------------------------------------------------------- rotation and cache write
// rope_kv_heads_kernel's way (pie_rope_kv.cu) over rows that each have a position and a slot of their own: a thread takes 8 pairs of features of one row for every HL-th
// head, 16 bytes an access, so a sine serves H / HL heads.  HBM-bound where there are many rows (8191 of 32 + 16 heads of 128 34.8 us, 5.8 TB/s), latency-bound where there
// are few (32 rows 3 us).
__global__ void __launch_bounds__(128) rope_kv_slots_kernel(uint16_t* q_out, uint16_t* kp, uint16_t* vp, long long tok_stride, long long head_stride, const RopeRows r,
                                                            const int32_t* positions, const int32_t* slots, const float* freqs, int rows, int n_slots, int Hq,
                                                            int Hkv, int D, int rest, int HL) {
  pdl_launch_dependents();
  pdl_wait();
  const int half = D / 2, PB = half / 8, pb = threadIdx.x % PB, rem = threadIdx.x / PB, hl = rem % HL;
  const int l = blockIdx.x * (128 / PB / HL) + rem / HL;
  if (l >= rows) return;
  const int slot = __ldg(slots + l);
  uint16_t* const qo = q_out + (size_t)l * Hq * D + pb * 8;
  if (slot < 0 || slot >= n_slots) {
    if (rest)
      for (int h = hl; h < Hq; h += HL)
        *reinterpret_cast<uint4*>(qo + (size_t)h * D) = *reinterpret_cast<uint4*>(qo + (size_t)h * D + half) = make_uint4(0, 0, 0, 0);
    return;
  }
  const float p = (float)__ldg(positions + l);
  float sn[8], cs[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rope_sincos(p * (1.0f / freqs[pb * 8 + e]), &sn[e], &cs[e]);
  const size_t at = (size_t)slot * tok_stride + pb * 8;
  // heads hl, hl + HL ...: the loads of four of them in flight before the first store
  auto heads = [&](const uint16_t* src, long long sh, uint16_t* dst, long long dh, int H, bool turn) {
    for (int h0 = hl; h0 < H; h0 += 4 * HL) {
      uint4 v1[4], v2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (h0 + i * HL < H) {
          const uint16_t* xr = src + (h0 + i * HL) * sh;
          v1[i] = *reinterpret_cast<const uint4*>(xr);
          v2[i] = *reinterpret_cast<const uint4*>(xr + half);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (h0 + i * HL >= H) break;
        if (turn) {
          const uint32_t a[4] = {v1[i].x, v1[i].y, v1[i].z, v1[i].w}, c[4] = {v2[i].x, v2[i].y, v2[i].z, v2[i].w};
          uint32_t r1[4], r2[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x1 = bf16lo(a[e]), y1 = bf16hi(a[e]), x2 = bf16lo(c[e]), y2 = bf16hi(c[e]);
            r1[e] = pack_bf16(__fsub_rn(__fmul_rn(x1, cs[2 * e]), __fmul_rn(x2, sn[2 * e])),
                              __fsub_rn(__fmul_rn(y1, cs[2 * e + 1]), __fmul_rn(y2, sn[2 * e + 1])));
            r2[e] = pack_bf16(__fadd_rn(__fmul_rn(x1, sn[2 * e]), __fmul_rn(x2, cs[2 * e])),
                              __fadd_rn(__fmul_rn(y1, sn[2 * e + 1]), __fmul_rn(y2, cs[2 * e + 1])));
          }
          v1[i] = make_uint4(r1[0], r1[1], r1[2], r1[3]);
          v2[i] = make_uint4(r2[0], r2[1], r2[2], r2[3]);
        }
        uint16_t* o = dst + (h0 + i * HL) * dh;
        *reinterpret_cast<uint4*>(o) = v1[i];
        *reinterpret_cast<uint4*>(o + half) = v2[i];
      }
    }
  };
  heads(r.q + l * r.qs.sl + pb * 8, r.qs.sh, qo, D, Hq, true);
  heads(r.k + l * r.ks.sl + pb * 8, r.ks.sh, kp + at, head_stride, Hkv, true);
  heads(r.v + l * r.vs.sl + pb * 8, r.vs.sh, vp + at, head_stride, Hkv, false);
}

}  // namespace pie

using namespace pie;

namespace {
bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
}  // namespace

extern "C" {

size_t pie_step_plan_words(const pie_step_dims* d) { return step_dims_status(d) ? 0 : (size_t)step_layout(*d).words; }

int pie_step_plan_offsets(const pie_step_dims* d, long long* o) {
  if (int s = step_dims_status(d)) return s;
  if (!o) return PIE_ENULL;
  const StepLayout l = step_layout(*d);
  const long long all[10] = {l.row_starts, l.contexts, l.sequences, l.positions, l.slots, l.block_table, l.logit_starts, l.logit_rows, l.draft_tokens, l.status};
  for (int i = 0; i < 10; ++i) o[i] = all[i];
  return PIE_OK;
}

int pie_step_plan_build(int32_t* plan, const pie_step_dims* d, const int32_t* token_ids, const int32_t* input_lengths, const int32_t* context_lengths,
                        const int32_t* draft_lengths, const int32_t* pages, long long n_page_ids, long long page_stride, void* stream) {
  if (int s = step_dims_status(d)) return s;
  if (!plan || !token_ids || !input_lengths || !context_lengths || (!pages && n_page_ids > 0)) return PIE_ENULL;
  if (n_page_ids < 0 || page_stride < 0) return PIE_EINVAL_SHAPE;
  if (off16(plan)) return PIE_EALIGN;
  PlanArgs a;
  a.plan = plan; a.d = *d; a.l = step_layout(*d);
  a.ids = token_ids; a.input = input_lengths; a.context = context_lengths; a.draft = draft_lengths; a.pages = pages;
  a.n_page_ids = n_page_ids; a.page_stride = page_stride;
  a.ctas = num_sms() < kStepMaxCtas ? num_sms() : kStepMaxCtas;
  const size_t smem = (size_t)(d->requests + 1) * (8 + 5 * 4);
  static std::atomic<unsigned long long> served{0};
  const cudaError_t set = once_per_device(served, [] {
    return cudaFuncSetAttribute(step_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kStepMaxRequests + 1) * (8 + 5 * 4));
  });
  if (set != cudaSuccess) return status_of(set);
  const long long cells = d->rows + (long long)d->requests * d->blocks + d->logit_rows + a.l.items;
  const long long grid = (cells + kPlanThreads - 1) / kPlanThreads;
  count_launch();
  return status_of(launch_pdl(step_plan_kernel, dim3((unsigned)(grid < a.ctas ? grid : a.ctas)), dim3(kPlanThreads), smem, (cudaStream_t)stream, a));
}

int pie_rope_kv_slots(void* q_out, void* kpool, void* vpool, const pie_kv_layout* kv, const pie_head_rows* q, const pie_head_rows* k, const pie_head_rows* v,
                      const int32_t* positions, const int32_t* slots, const float* freqs, int rows, int pages, int Hq, int Hkv, int D, int rest, void* stream) {
  if (rows == 0) return PIE_OK;
  if (!q_out || !kpool || !vpool || !kv || !q || !k || !v || !q->p || !k->p || !v->p || !positions || !slots || !freqs) return PIE_ENULL;
  if (rows < 0 || pages <= 0 || Hq <= 0 || Hkv <= 0 || (D != 64 && D != 128) || kv->tok_stride <= 0 || kv->tok_stride % 8 || kv->head_stride % 8 ||
      (long long)pages * kStepPage > 0x7fffffff)
    return PIE_EINVAL_SHAPE;
  RopeRows r;
  const pie_head_rows* src[3] = {q, k, v};
  const uint16_t** at[3] = {&r.q, &r.k, &r.v};
  KvSrc* st[3] = {&r.qs, &r.ks, &r.vs};
  for (int i = 0; i < 3; ++i) {
    if (src[i]->stride_h % 8 || src[i]->stride_l % 8) return PIE_EINVAL_SHAPE;
    if (off16(src[i]->p)) return PIE_EALIGN;
    *at[i] = (const uint16_t*)src[i]->p;
    *st[i] = {0, src[i]->stride_h, src[i]->stride_l};
  }
  if (off16(q_out) || off16(kpool) || off16(vpool)) return PIE_EALIGN;
  const int lanes = 128 / (D / 16), HL = rows >= 1024 ? 4 : lanes, per = lanes / HL;
  count_launch();
  return status_of(launch_pdl(rope_kv_slots_kernel, dim3((unsigned)((rows + per - 1) / per)), dim3(128), 0, (cudaStream_t)stream, (uint16_t*)q_out, (uint16_t*)kpool,
                              (uint16_t*)vpool, kv->tok_stride, kv->head_stride, r, positions, slots, freqs, rows, pages * kStepPage, Hq, Hkv, D, rest, HL));
}

}  // extern "C"
