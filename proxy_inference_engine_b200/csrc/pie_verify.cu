// Drafted tokens against the target's probabilities (include/pie_b200.h has the definition), on the device: no counterpart in the reference, whose engine decodes one
// token a step (PIE/engine/inference_engine.py:259-297); the log-probabilities are its own, f32(logits) - logsumexp (:268-269), at the temperature of the draw.
//
// Two launches.  verify_stats_kernel reads every row of logits once: maximum and sum of exponentials (greedy: and the first largest) of slices, in 32 bits.
// verify_emit_kernel: each CTA of a request joins its rows' slices, finds how many drafted tokens are accepted, and takes a slice of the vocabulary of the one row behind
// them; the last CTA to finish joins the slices' best.  All of it is bound by HBM: a row of 128256 logits is 257 KB.
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
  float itemp;                      // 1 / temp; greedy: 1
  int greedy;
  const float *uniforms, *noise;
  int splits, emit_splits;          // slices of a row in either launch
  float* stats;                     // [rows][2][splits][4]: maximum, sum of exp, index of the maximum (greedy)
  unsigned long long* best;         // [requests][emit_splits]
  unsigned int* count;              // [requests], zero between launches
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
// (m, s) <- the maximum and the sum of exponentials of two parts
__device__ __forceinline__ void ver_join(float& m, float& s, float m2, float s2) {
  const float mx = fmaxf(m, m2);
  s = (s == 0.f ? 0.f : s * __expf(m - mx)) + (s2 == 0.f ? 0.f : s2 * __expf(m2 - mx));
  m = mx;
}
// elements [lo, hi) of slice i of n
__device__ __forceinline__ void ver_slice(int vocab, int i, int n, int& lo, int& hi) {
  const int per = ((vocab + n - 1) / n + 7) / 8 * 8;
  lo = min(i * per, vocab);
  hi = min(lo + per, vocab);
}

__global__ void __launch_bounds__(kVerThreads) verify_stats_kernel(const __grid_constant__ VerArgs a) {
  __shared__ float sm[kVerThreads / 32][2];
  __shared__ unsigned long long km[kVerThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
  const uint16_t* x = (which ? a.guess : a.logits) + (size_t)r * a.ld;
  int lo, hi;
  ver_slice(a.vocab, blockIdx.x, a.splits, lo, hi);
  float m = -INFINITY, s = 0.f;
  unsigned long long key = 0;
  for (int i = lo + tid; i < hi; i += kVerThreads) {
    const float v = bf16lo((uint32_t)__ldg(x + i)) + 0.f;   // (-0 is 0)
    if (a.greedy && v == v) key = ver_max(key, ver_key(v, i));
    const float t = v * a.itemp;
    if (t > m) { s = s * __expf(m - t) + 1.f; m = t; }
    else if (t != -INFINITY) s += __expf(t - m);   // (a NaN ends up in the sum)
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    ver_join(m, s, m2, s2);
  }
  if ((tid & 31) == 0) { sm[tid >> 5][0] = m; sm[tid >> 5][1] = s; }
  if (a.greedy) key = ver_block_max(key, km); else __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kVerThreads / 32; ++w) ver_join(m, s, sm[w][0], sm[w][1]);
    *reinterpret_cast<float4*>(a.stats + (((size_t)r * 2 + which) * a.splits + blockIdx.x) * 4) =
        make_float4(m, s, __uint_as_float((uint32_t)(key >> 32)), __int_as_float(key ? ver_index(key) : 0));
  }
}

__global__ void __launch_bounds__(kVerThreads) verify_emit_kernel(const __grid_constant__ VerArgs a) {
  __shared__ float lse[2][kVerMaxDraft + 1];
  __shared__ int top[kVerMaxDraft + 1], ok[kVerMaxDraft + 1], s_accepted, s_last;
  __shared__ unsigned long long km[kVerThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const int s = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
    float l[2] = {0.f, 0.f};
    unsigned long long key = 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which && (!a.guess || last)) break;
      float m = -INFINITY, sum = 0.f;
      for (int i = lane; i < a.splits; i += 32) {
        const float4 p = __ldcg(reinterpret_cast<const float4*>(a.stats + (((size_t)r * 2 + which) * a.splits + i) * 4));
        ver_join(m, sum, p.x, p.y);
        if (!which) key = ver_max(key, ((unsigned long long)__float_as_uint(p.z) << 32) | (uint32_t)~__float_as_int(p.w));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, sum, o);
        ver_join(m, sum, m2, s2);
        key = ver_max(key, __shfl_xor_sync(0xffffffffu, key, o));
      }
      l[which] = m + logf(sum);
    }
    if (lane == 0) {
      lse[0][j] = l[0];
      lse[1][j] = l[1];
      top[j] = key >> 32 ? ver_index(key) : 0;
      bool yes = !last && real;
      if (yes && a.greedy) yes = top[j] == x;
      else if (yes) {
        const float p = expf(bf16lo((uint32_t)a.logits[(size_t)r * a.ld + x]) * a.itemp - l[0]);
        const float q = a.guess ? expf(bf16lo((uint32_t)a.guess[(size_t)r * a.ld + x]) * a.itemp - l[1]) : 1.f;
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
    const float lp = lse[0][k], lq = lse[1][k];
    auto race = [&](int lo, int hi, bool whole) {
      unsigned long long key = 0;
      for (int i = lo + tid; i < hi; i += kVerThreads) {
        float w = expf(bf16lo((uint32_t)__ldg(x + i)) * a.itemp - lp);
        if (!whole) {
          if (g) w -= expf(bf16lo((uint32_t)__ldg(g + i)) * a.itemp - lq);
          if (i == out) w = 0.f;
        }
        if (w > 0.f) key = ver_max(key, ver_key(w / -logf(__ldg(u + i)), i));
      }
      return ver_block_max(key, km);
    };
    int lo, hi;
    ver_slice(a.vocab, blockIdx.x, a.emit_splits, lo, hi);
    unsigned long long key = race(lo, hi, false);
    if (a.emit_splits > 1) {
      if (tid == 0) {
        __stcg(a.best + (size_t)s * a.emit_splits + blockIdx.x, key);
        unsigned int before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.count + s) : "memory");
        s_last = before == (unsigned)a.emit_splits - 1;
        if (s_last) a.count[s] = 0;
      }
      __syncthreads();
      if (!s_last) return;
      key = 0;
      for (int i = tid; i < a.emit_splits; i += kVerThreads) key = ver_max(key, __ldcg(a.best + (size_t)s * a.emit_splits + i));
      key = ver_block_max(key, km);
    }
    if (key == 0 && refused) key = race(0, a.vocab, true);
    token = key ? ver_index(key) : 0;
  }
  for (int j = tid; j <= a.most; j += kVerThreads) {
    int t = -1;
    float lp = 0.f;
    if (j <= k) {
      t = j < k ? __ldg(a.draft + r0 + j) : token;
      lp = bf16lo((uint32_t)a.logits[(size_t)(r0 + j) * a.ld + t]) * a.itemp - lse[0][j];
    }
    tokens[j] = t;
    logprobs[j] = lp;
  }
  if (tid == 0) a.counts[s] = k + 1;
}

struct VerPlan { int splits, emit_splits; size_t stats, best, bytes; };
static VerPlan ver_plan(int requests, int rows, int vocab) {
  VerPlan p;
  // slices of at least 4096 tokens, as many as give the device two rounds of CTAs
  auto pick = [&](int units) {
    const int most = (vocab + 4095) / 4096, want = (4 * 148 + units - 1) / units;
    return want < 1 ? 1 : want > most ? (most < kVerMaxSplits ? most : kVerMaxSplits) : want < kVerMaxSplits ? want : kVerMaxSplits;
  };
  p.splits = pick(rows);
  p.emit_splits = pick(requests);
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
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return PIE_EALIGN;
  VerArgs a;
  a.tokens = tokens; a.counts = counts; a.logprobs = logprobs;
  a.logits = (const uint16_t*)logits; a.guess = (const uint16_t*)draft_logits; a.ld = ld;
  a.draft = draft_tokens; a.starts = logit_starts;
  a.requests = requests; a.rows = rows; a.vocab = vocab; a.most = max_draft;
  a.greedy = temp == 0.f; a.itemp = a.greedy ? 1.f : 1.f / temp;
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
