// Drafted tokens against the target's probabilities (include/pie_b200.h has the definition), on the device: no counterpart in the reference, whose engine decodes one
// token a step (PIE/engine/inference_engine.py:259-297); the log-probabilities are its own, f32(logits) - logsumexp (:268-269), at the temperature of the draw.
//
// Two launches.  verify_stats_kernel reads every row of logits once: maximum and sum of exponentials (greedy: and the first largest) of slices, in 32 bits.
// verify_emit_kernel: each CTA of a request joins its rows' slices, finds how many drafted tokens are accepted, and takes slices of the one row behind them through the race for
// its token; the last CTA to finish joins the slices' best.  (The joining by the last CTA of the first launch, once for a request, cost more in its tail than it saved: 39 -> 46 us.)
// A row of 128256 logits is 257 KB: HBM at the least, but it gives 1.3 to 3.8 TB/s, and the issue slots are 27 to 42 % active: what bounds is latency.  A CTA's start and end are as long as its
// slice, and a turn of the race uses its loads at once, between barriers.  Device time in a captured row of such calls, inputs not in L2: 5 rows greedy 5.5 us, 16 x 8 13.0, 32 x 6 looked-up
// drafts 22.0, 64 x 6 rows against a drafter's 40.4 (3.1 TB/s).
#include <algorithm>

#include "pie_internal.h"
#include "pie_ptx.cuh"

namespace pie {

constexpr int kVerThreads = 256, kVerMaxDraft = 127, kVerMaxSplits = 64;

struct VerArgs {
  int32_t* tokens;
  int32_t* counts;
  float* logprobs;
  const uint16_t *logits, *guess;   // guess: the draft's logits, or nullptr
  long long ld;
  const int32_t *draft, *starts;
  int requests, rows, vocab, most;
  float itemp;                      // 1 / temp, at most 2^125 (times log2(e) it is finite); greedy: 1
  int greedy;
  const float *uniforms, *noise;
  int splits, emit_splits;          // slices of a row in either launch
  float* stats;                     // [rows][2][splits][4]: maximum, sum of exp, index of the maximum (greedy)
  unsigned long long* best;         // [requests][emit_splits]
  unsigned int* count;              // [requests], set to zero by the first launch for the second
};

// larger keys are larger scores, of equal scores the lower index; 0: none
__device__ __forceinline__ unsigned long long ver_key(float score, int index) {
  const uint32_t u = __float_as_uint(score), k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)k << 32) | (uint32_t)~index;
}
__device__ __forceinline__ int ver_index(unsigned long long key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ unsigned long long ver_max(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned long long ver_block_max(unsigned long long v, unsigned long long* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = ver_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kVerThreads / 32; ++w) v = ver_max(v, sm[w]);
  __syncthreads();
  return v;
}
// (m, s) <- the maximum and the sum of exp2(c (x - maximum)) of two parts
__device__ __forceinline__ void ver_join(float& m, float& s, float m2, float s2, float c) {
  const float mx = fmaxf(m, m2);
  s = (s == 0.f ? 0.f : s * exp2f((m - mx) * c)) + (s2 == 0.f ? 0.f : s2 * exp2f((m2 - mx) * c));
  m = mx;
}
// A row is read 16 bytes (8 logits) at a time from its first 16-byte boundary on; what lies in front of that and behind the last whole 8 is few single ones.
struct VerRow {
  const uint16_t* x;
  int head, vectors, tail;   // logits in front, 8 at a time, first one behind
};
__device__ __forceinline__ VerRow ver_row(const uint16_t* x, int vocab) {
  VerRow r;
  r.x = x;
  r.head = min((int)((8 - ((reinterpret_cast<uintptr_t>(x) >> 1) & 7)) & 7), vocab);
  r.vectors = (vocab - r.head) / 8;
  r.tail = r.head + 8 * r.vectors;
  return r;
}
// vectors [lo, hi) of slice i of n, whole turns of the CTA
constexpr int kVerTurn = 4;   // vectors a thread takes at a time
__device__ __forceinline__ void ver_slice(int vectors, int i, int n, int& lo, int& hi) {
  const int per = (vectors + n * kVerTurn * kVerThreads - 1) / (n * kVerTurn * kVerThreads) * (kVerTurn * kVerThreads);
  lo = min(i * per, vectors);
  hi = min(lo + per, vectors);
}
__device__ __forceinline__ uint4 ver_load(const uint16_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ uint32_t ver_max2(uint32_t a, uint32_t b) {   // of two pairs of bf16; a number before a NaN
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ float ver_exp2(float x) {   // results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float ver_warp_max(float x) {   // of numbers, by integers in their order
  const int i = __float_as_int(x), v = __reduce_max_sync(0xffffffffu, i ^ ((i >> 31) & 0x7fffffff));
  return __int_as_float(v ^ ((v >> 31) & 0x7fffffff));
}
// A thread's part of a row: maximum x and sum of exp2(c x + off), off = -c maximum rounded -- one fused multiply-add an exponential, and what the rounding does to all
// of them alike (2^-24 of c x, more than a sum may be off by) is taken back at the end.  Where it would do too much (steep: a maximum of thousands at an ordinary
// temperature, a slice of nothing but the type's lowest value, a temperature near 0) the sum is of exp2(c (x - maximum)), an operation more.  32 logits a turn; their
// maximum is taken in pairs of bf16, and moves the sum once a turn.  Greedy: where it moves is where the first largest lies so far.
struct VerSum {
  float m = -INFINITY, off = 0.f, s = 0.f;
  int index = -1;
  __device__ __forceinline__ bool steep() const { return fabsf(off) > 16384.f; }   // (at the border the factor is 2^(2^-11))
  __device__ __forceinline__ float term(float x, float c) const { return x == -INFINITY ? 0.f : ver_exp2(steep() ? (x - m) * c : fmaf(x, c, off)); }
  __device__ __forceinline__ void move(float mx, float c) {
    const float to = -mx * c;
    if (m != -INFINITY) {                                    // (a NaN in s stays one)
      if (fmaxf(fabsf(to), fabsf(off)) <= 16384.f) s *= ver_exp2(to - off);
      else s = sum(c) * ver_exp2((m - mx) * c) * (fabsf(to) > 16384.f ? 1.f : ver_exp2(fmaf(mx, c, to)));
    }
    m = mx;
    off = to;
  }
  __device__ __forceinline__ void one(float x, int i, float c) {
    x += 0.f;                                                // (-0 is 0)
    if (x > m) { move(x, c); index = i; }
    if (index < 0 && x == x) index = i;
    s += term(x, c);
  }
  __device__ __forceinline__ float sum(float c) const { return m == -INFINITY || steep() ? s : s * ver_exp2(-fmaf(m, c, off)); }   // of exp2(c (x - m))
};

// two fp32 operations an instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 v2_pack(float a, float b) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void v2_unpack(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 v2_fma(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 v2_add(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__global__ void __launch_bounds__(kVerThreads) verify_stats_kernel(const __grid_constant__ VerArgs a) {
  __shared__ float sm[kVerThreads / 32][2];
  __shared__ unsigned long long km[kVerThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
  // (Here, and not by the last CTA to count: where the counters lie depends on the call, and a call of another shape may have left numbers there.)
  if (a.emit_splits > 1 && blockIdx.x == 0 && r == 0 && !which)
    for (int i = tid; i < a.requests; i += kVerThreads) a.count[i] = 0;
  if (which) {   // a request's last row judges no token: its draft's logits are not read
    // (Where starts do not rise, another request may judge its token all the same: by a sum of 0 it refuses it.  Said ahead of the look at them, which costs the others no registers.)
    if (tid == 0) *reinterpret_cast<float2*>(a.stats + (((size_t)r * 2 + 1) * a.splits + blockIdx.x) * 4) = make_float2(-INFINITY, 0.f);
    bool last = false;
    for (int i = tid; i < a.requests; i += kVerThreads) last = last || __ldg(a.starts + i + 1) == r + 1;
    if (__syncthreads_or(last)) return;
  }
  const VerRow row = ver_row((which ? a.guess : a.logits) + (size_t)r * a.ld, a.vocab);
  const float c = a.itemp * 1.4426950408889634f;
  VerSum sum;
  if (blockIdx.x == 0 && tid < row.head) sum.one(bf16lo((uint32_t)__ldg(row.x + tid)), tid, c);
  int lo, hi;
  ver_slice(row.vectors, blockIdx.x, a.splits, lo, hi);
  uint4 x[kVerTurn];
  auto load = [&](int v0) {
#pragma unroll
    for (int t = 0; t < kVerTurn; ++t) {
      const int v = v0 + t * kVerThreads;
      x[t] = v < hi ? ver_load(row.x + row.head + 8 * (size_t)v) : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);   // -inf
    }
  };
  load(lo + tid);
  for (int v0 = lo + tid; v0 < hi; v0 += kVerTurn * kVerThreads) {
    uint32_t w[kVerTurn][4];
#pragma unroll
    for (int t = 0; t < kVerTurn; ++t) { w[t][0] = x[t].x; w[t][1] = x[t].y; w[t][2] = x[t].z; w[t][3] = x[t].w; }
    load(v0 + kVerTurn * kVerThreads);
    uint32_t m2 = w[0][0];
#pragma unroll
    for (int t = 0; t < kVerTurn; ++t) m2 = ver_max2(ver_max2(m2, ver_max2(w[t][0], w[t][1])), ver_max2(w[t][2], w[t][3]));
    const float mx = fmaxf(bf16lo(m2), bf16hi(m2)) + 0.f;
    if (mx > sum.m || (a.greedy && sum.index < 0)) {
      if (mx > sum.m) { sum.move(mx, c); sum.index = -1; }
      if (a.greedy) {   // the first of this turn that is the largest so far
#pragma unroll
        for (int t = 0; t < kVerTurn; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float f = (e & 1 ? bf16hi(w[t][e / 2]) : bf16lo(w[t][e / 2])) + 0.f;
            if (sum.index < 0 && f == sum.m && v0 + t * kVerThreads < hi) sum.index = row.head + 8 * (v0 + t * kVerThreads) + e;
          }
      }
    }
    if (sum.steep()) {
#pragma unroll 1
      for (int t = 0; t < kVerTurn; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t pair = t == 0 ? w[0][e] : t == 1 ? w[1][e] : t == 2 ? w[2][e] : w[3][e];
          sum.s += sum.term(bf16lo(pair), c) + sum.term(bf16hi(pair), c);
        }
      continue;
    }
    const f32x2 c2 = v2_pack(c, c), off2 = v2_pack(sum.off, sum.off);
    f32x2 s01 = v2_pack(0.f, 0.f), s23 = s01;
#pragma unroll
    for (int t = 0; t < kVerTurn; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float y0, y1;
        v2_unpack(v2_fma(v2_pack(bf16lo(w[t][e]), bf16hi(w[t][e])), c2, off2), y0, y1);
        const f32x2 y = v2_pack(ver_exp2(y0), ver_exp2(y1));
        if (e & 1) s23 = v2_add(s23, y);
        else s01 = v2_add(s01, y);
      }
    float s0, s1;
    v2_unpack(v2_add(s01, s23), s0, s1);
    sum.s += s0 + s1;
  }
  if ((int)blockIdx.x == a.splits - 1 && tid < a.vocab - row.tail) sum.one(bf16lo((uint32_t)__ldg(row.x + row.tail + tid)), row.tail + tid, c);
  const unsigned long long mine = a.greedy && sum.index >= 0 ? ver_key(sum.m, sum.index) : 0;
  const float m = ver_warp_max(sum.m), part = sum.sum(c);
  float s = part == 0.f ? 0.f : part * exp2f((sum.m - m) * c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) { sm[tid >> 5][0] = m; sm[tid >> 5][1] = s; }
  unsigned long long key = 0;
  if (a.greedy) key = ver_block_max(mine, km); else __syncthreads();
  if (tid == 0) {
    float mb = m, sb = s;
    for (int w = 1; w < kVerThreads / 32; ++w) ver_join(mb, sb, sm[w][0], sm[w][1], c);
    *reinterpret_cast<float4*>(a.stats + (((size_t)r * 2 + which) * a.splits + blockIdx.x) * 4) =
        make_float4(mb, sb, __uint_as_float((uint32_t)(key >> 32)), __int_as_float(key ? ver_index(key) : 0));
  }
}

__global__ void __launch_bounds__(kVerThreads) verify_emit_kernel(const __grid_constant__ VerArgs a) {
  __shared__ float2 dist[2][kVerMaxDraft + 1];   // of p and q of each row: maximum, sum of exp2(c (x - maximum))
  __shared__ int top[kVerMaxDraft + 1], ok[kVerMaxDraft + 1], s_accepted, s_last, s_best;
  __shared__ unsigned long long km[kVerThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float c = a.itemp * 1.4426950408889634f;
  const int r0 = max(0, min(__ldg(a.starts + s), a.rows)), r1 = max(r0, min(__ldg(a.starts + s + 1), a.rows));
  const int n = min(r1 - r0, a.most + 1);   // rows that count
  int32_t* const tokens = a.tokens + (size_t)s * (a.most + 1);
  float* const logprobs = a.logprobs + (size_t)s * (a.most + 1);
  if (n == 0) {
    if (blockIdx.x == 0) {
      for (int j = tid; j <= a.most; j += kVerThreads) { tokens[j] = -1; logprobs[j] = 0.f; }
      if (tid == 0) a.counts[s] = 0;
    }
    return;
  }
  // ---- a warp a row: its logarithm of the sum, its largest, and whether its token is accepted
  for (int j = warp; j < n; j += kVerThreads / 32) {
    const int r = r0 + j, x = __ldg(a.draft + r);
    const bool last = j == n - 1, real = x >= 0 && x < a.vocab;
    float2 d[2] = {{0.f, 1.f}, {0.f, 1.f}};
    unsigned long long key = 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which && (!a.guess || last)) break;
      float m = -INFINITY, sum = 0.f;
      for (int i = lane; i < a.splits; i += 32) {
        const float4 p = __ldcg(reinterpret_cast<const float4*>(a.stats + (((size_t)r * 2 + which) * a.splits + i) * 4));
        ver_join(m, sum, p.x, p.y, c);
        if (!which) key = ver_max(key, ((unsigned long long)__float_as_uint(p.z) << 32) | (uint32_t)~__float_as_int(p.w));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
        ver_join(m, sum, m2, s2, c);
        key = ver_max(key, __shfl_xor_sync(0xffffffffu, key, o));
      }
      d[which] = make_float2(m, sum);
    }
    if (lane == 0) {
      dist[0][j] = d[0];
      dist[1][j] = d[1];
      top[j] = key >> 32 ? ver_index(key) : 0;
      bool yes = !last && real;
      if (yes && a.greedy) yes = top[j] == x;
      else if (yes) {
        const float p = expf((bf16lo((uint32_t)a.logits[(size_t)r * a.ld + x]) - d[0].x) * a.itemp) / d[0].y;
        const float q = a.guess ? expf((bf16lo((uint32_t)a.guess[(size_t)r * a.ld + x]) - d[1].x) * a.itemp) / d[1].y : 1.f;
        yes = a.uniforms[r] * q < p;
      }
      ok[j] = yes;
    }
  }
  __syncthreads();
  if (tid == 0) {
    int k = 0;
    while (k < n - 1 && ok[k]) ++k;
    s_accepted = k;
  }
  __syncthreads();
  const int k = s_accepted, r = r0 + k;
  const uint16_t* const x = a.logits + (size_t)r * a.ld;
  int token;
  if (a.greedy) {
    token = top[k];
  } else {
    const bool refused = k < n - 1;
    const uint16_t* const g = refused && a.guess ? a.guess + (size_t)r * a.ld : nullptr;
    const int out = refused && !a.guess ? __ldg(a.draft + r) : -1;   // the token that was refused
    const float* const u = a.noise + (size_t)s * a.vocab;
    // p = exp2(c (x - maximum)) / sum
    const float2 dp = dist[0][k], dq = dist[1][k];
    const float kp = 1.f / dp.y, kq = 1.f / dq.y;
    const VerRow row = ver_row(x, a.vocab);
    const bool flat = !(reinterpret_cast<uintptr_t>(u + row.head) & 15);   // the draws can be read 16 bytes at a time as well
    // The race: of weights w and draws u, the largest w / E, E = -log(u), over turns i, i + n, ... of the row; whole: of the target's own weights.
    // 1 - u <= E <= (1 - u) / u, so with b = w / (1 - u) a token's score lies between b u and b, which near u = 1, where the winners lie, is as good as equal: a thread keeps
    // the b of its 32 tokens, the CTA the largest b u, and logarithms are taken of the one or two whose b is not below that.  (E by logf: near u = 1 it is good to its last
    // place, and the approximation unit's is not.  A logarithm for each token, 64 requests: 36 us.)
    auto race = [&](int i, int n, bool whole) {
      const uint16_t* const q = whole ? nullptr : g;
      const int not_this = whole ? -1 : out;
      unsigned long long key = 0;
      auto weight = [&](float xi, float qi) {
        float w = __fmul_rn(ver_exp2((xi - dp.x) * c), kp);
        if (q) w = __fsub_rn(w, __fmul_rn(ver_exp2((qi - dq.x) * c), kq));   // (no fused form: p = q leaves nothing)
        return w;
      };
      auto run = [&](int at) {   // exactly
        const float w = at == not_this ? 0.f : weight(bf16lo((uint32_t)__ldg(x + at)), q ? bf16lo((uint32_t)__ldg(q + at)) : 0.f);
        const float e = fmaxf(-logf(fmaxf(__ldg(u + at), 1.17549435e-38f)), 0.f);   // (a draw of 0 is the smallest there is: a token that is alone wins with it)
        if (w > 0.f) key = ver_max(key, ver_key(w / e, at));
      };
      const int ends = row.head + a.vocab - row.tail;   // (at most 14)
      if (i == 0 && tid < ends) run(tid < row.head ? tid : row.tail + tid - row.head);
      for (int v0 = i * kVerTurn * kVerThreads; v0 < row.vectors; v0 += n * kVerTurn * kVerThreads) {
        float bound[8 * kVerTurn], least = 0.f, most = 0.f;   // of a token without weight (or with a NaN): 0, as of one that is not there
#pragma unroll
        for (int t = 0; t < kVerTurn; ++t) {
          const int v = v0 + t * kVerThreads + tid, at = row.head + 8 * v;
          if (v >= row.vectors) {
#pragma unroll
            for (int e = 0; e < 8; ++e) bound[8 * t + e] = 0.f;
            continue;
          }
          const uint4 xv = ver_load(x + at), qv = q ? ver_load(q + at) : make_uint4(0, 0, 0, 0);
          float ui[8];
          if (flat) {
            *reinterpret_cast<float4*>(ui) = __ldg(reinterpret_cast<const float4*>(u + at));
            *reinterpret_cast<float4*>(ui + 4) = __ldg(reinterpret_cast<const float4*>(u + at + 4));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) ui[e] = __ldg(u + at + e);
          }
          const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w}, qw[4] = {qv.x, qv.y, qv.z, qv.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float r;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f - ui[e]));   // (a draw of 1: infinite, and looked at)
            float b = fmaxf(weight(e & 1 ? bf16hi(xw[e / 2]) : bf16lo(xw[e / 2]), e & 1 ? bf16hi(qw[e / 2]) : bf16lo(qw[e / 2])), 0.f) * r;
            if (at + e == not_this) b = 0.f;
            bound[8 * t + e] = b;
            least = fmaxf(least, b * ui[e]);
            most = fmaxf(most, b);
          }
        }
        if (tid == 0) s_best = 0;
        __syncthreads();
        const int mine = __reduce_max_sync(0xffffffffu, __float_as_int(least));   // (none is negative: in the order of their bits)
        if (lane == 0) atomicMax(&s_best, mine);
        __syncthreads();
        const float bar = __int_as_float(s_best) * 0.99999f;
        if (most >= bar && most > 0.f) {
          unsigned left = 0;
#pragma unroll
          for (int e = 0; e < 8 * kVerTurn; ++e) left |= (unsigned)(bound[e] >= bar && bound[e] > 0.f) << e;
          for (; left; left &= left - 1) {
            const int e = __ffs(left) - 1;
            run(row.head + 8 * (v0 + (e / 8) * kVerThreads + tid) + e % 8);
          }
        }
        __syncthreads();
      }
      return ver_block_max(key, km);
    };
    unsigned long long key = race(blockIdx.x, a.emit_splits, false);
    if (a.emit_splits > 1) {
      if (tid == 0) {
        __stcg(a.best + (size_t)s * a.emit_splits + blockIdx.x, key);
        unsigned int before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.count + s) : "memory");
        s_last = before == (unsigned)a.emit_splits - 1;
      }
      __syncthreads();
      if (!s_last) return;
      key = 0;
      for (int i = tid; i < a.emit_splits; i += kVerThreads) key = ver_max(key, __ldcg(a.best + (size_t)s * a.emit_splits + i));
      key = ver_block_max(key, km);
    }
    if (key == 0 && refused) key = race(0, 1, true);
    token = key ? ver_index(key) : 0;
  }
  for (int j = tid; j <= a.most; j += kVerThreads) {
    int t = -1;
    float lp = 0.f;
    if (j <= k) {
      t = j < k ? __ldg(a.draft + r0 + j) : token;
      lp = (bf16lo((uint32_t)a.logits[(size_t)(r0 + j) * a.ld + t]) - dist[0][j].x) * a.itemp - logf(dist[0][j].y);
    }
    tokens[j] = t;
    logprobs[j] = lp;
  }
  if (tid == 0) a.counts[s] = k + 1;
}

struct VerPlan { int splits, emit_splits; size_t stats, best, bytes; };
static VerPlan ver_plan(int requests, int rows, int vocab) {
  VerPlan p;
  // as many slices of a row as give every SM some CTAs, all of the same power of two of turns but the last
  auto pick = [&](int units, int want) {
    const int turns = (vocab / 8 + kVerTurn * kVerThreads - 1) / (kVerTurn * kVerThreads);
    const long long most = std::max(1LL, (long long)turns * units / (want * num_sms()));
    long long per = 1;
    while (2 * per <= most || (turns + per - 1) / per > kVerMaxSplits) per *= 2;
    return (int)std::max(1LL, (turns + per - 1) / per);
  };
  p.splits = pick(rows, 4);
  p.emit_splits = pick(requests, 3);
  const size_t counts = ((size_t)requests * 4 + 255) & ~(size_t)255;
  p.stats = counts;
  p.best = p.stats + (size_t)rows * 2 * p.splits * 16;
  p.bytes = p.best + (size_t)requests * p.emit_splits * 8;
  return p;
}

}  // namespace pie

using namespace pie;

extern "C" {

size_t pie_verify_workspace_bytes(int requests, int rows, int vocab) {
  return requests <= 0 || rows <= 0 || vocab <= 0 ? 0 : ver_plan(requests, rows, vocab).bytes;
}

int pie_verify_draft(int32_t* tokens, int32_t* counts, float* logprobs, const void* logits, const void* draft_logits, long long ld, const int32_t* draft_tokens,
                     const int32_t* logit_starts, int requests, int rows, int vocab, int max_draft, float temp, const float* uniforms, const float* noise,
                     void* workspace, size_t workspace_bytes, void* stream) {
  if (requests == 0) return PIE_OK;
  if (!tokens || !counts || !logprobs || !logits || !draft_tokens || !logit_starts) return PIE_ENULL;
  if (requests < 0 || requests > 65535 || rows <= 0 || rows > 65535 || vocab <= 0 || ld < vocab || max_draft < 0 || max_draft > kVerMaxDraft) return PIE_EINVAL_SHAPE;
  if (!(temp >= 0.f) || temp > 3.4028234e38f) return PIE_EINVAL_SHAPE;
  if (temp > 0.f ? !uniforms || !noise : draft_logits != nullptr) return temp > 0.f ? PIE_ENULL : PIE_EINVAL_SHAPE;
  const VerPlan p = ver_plan(requests, rows, vocab);
  if (!workspace || workspace_bytes < p.bytes) return PIE_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(draft_logits)) & 15) return PIE_EALIGN;
  VerArgs a;
  a.tokens = tokens; a.counts = counts; a.logprobs = logprobs;
  a.logits = (const uint16_t*)logits; a.guess = (const uint16_t*)draft_logits; a.ld = ld;
  a.draft = draft_tokens; a.starts = logit_starts;
  a.requests = requests; a.rows = rows; a.vocab = vocab; a.most = max_draft;
  a.greedy = temp == 0.f; a.itemp = a.greedy ? 1.f : std::min(1.f / temp, 4.25352959e37f);
  a.uniforms = uniforms; a.noise = noise;
  a.splits = p.splits; a.emit_splits = a.greedy ? 1 : p.emit_splits;
  uint8_t* const ws = (uint8_t*)workspace;
  a.count = (unsigned int*)ws; a.stats = (float*)(ws + p.stats); a.best = (unsigned long long*)(ws + p.best);
  count_launch(2);
  cudaError_t e = launch_pdl(verify_stats_kernel, dim3(a.splits, rows, draft_logits ? 2 : 1), dim3(kVerThreads), 0, (cudaStream_t)stream, a);
  if (e == cudaSuccess) e = launch_pdl(verify_emit_kernel, dim3(a.emit_splits, requests), dim3(kVerThreads), 0, (cudaStream_t)stream, a);
  return status_of(e);
}

}  // extern "C"
