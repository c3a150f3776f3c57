// Causal attention of every request's new tokens over its pages (include/pie_b200.h): a warp per (row, query head), the keys one by one with a running maximum and sum.
// Replaces, for the rows of a ragged step, mx.fast.scaled_dot_product_attention with the causal mask of create_attention_mask (PIE/models/base.py:18-53, 92-113).
#include "pie_ptx.cuh"
#include "pie_step_plan.h"

namespace pie {

struct ChunkArgs {
  uint16_t* out;
  const uint16_t *q, *k, *v;
  long long q_row, q_head, tok, head;
  const int32_t* plan;
  StepLayout l;
  pie_step_dims d;
  float scale_log2e;
  int rest;
};

template <int D>
__global__ void __launch_bounds__(128) chunk_attn_kernel(const __grid_constant__ ChunkArgs a) {
  constexpr int E = D / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= a.d.Hq) return;
  uint16_t* const o = a.out + ((size_t)t * a.d.Hq + h) * D;
  const int s = a.plan[a.l.sequences + t];
  if (s < 0) {
    if (a.rest)
      for (int e = 0; e < E; ++e) o[32 * e + lane] = 0;
    return;
  }
  const int last = a.plan[a.l.positions + t], kvh = h / (a.d.Hq / a.d.Hkv);
  const int32_t* const table = a.plan + a.l.block_table + (size_t)s * a.d.blocks;
  float q[E], acc[E], m = -INFINITY, sum = 0.f;
  for (int e = 0; e < E; ++e) { q[e] = bf16lo((uint32_t)a.q[t * a.q_row + h * a.q_head + 32 * e + lane]) * a.scale_log2e; acc[e] = 0.f; }
  for (int j = 0; j <= last; ++j) {
    const size_t at = ((size_t)table[j / kStepPage] * kStepPage + j % kStepPage) * a.tok + kvh * a.head;
    float x = 0.f;
    for (int e = 0; e < E; ++e) x += q[e] * bf16lo((uint32_t)a.k[at + 32 * e + lane]);
    x = warp_sum(x);
    const float mx = fmaxf(m, x), f = m == -INFINITY ? 0.f : exp2f(m - mx), p = exp2f(x - mx);
    sum = sum * f + p;
    m = mx;
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * f + p * bf16lo((uint32_t)a.v[at + 32 * e + lane]);
  }
  for (int e = 0; e < E; ++e) o[32 * e + lane] = f2bf(acc[e] / sum);
}

}  // namespace pie

using namespace pie;

extern "C" {

size_t pie_chunk_attn_workspace_bytes(const pie_step_dims* d, int D) { return step_dims_status(d) || (D != 64 && D != 128) ? 0 : 256; }

int pie_chunk_attn(void* out, const pie_head_rows* q, const void* kpool, const void* vpool, const pie_kv_layout* kv, const int32_t* plan, const pie_step_dims* d, int D,
                   float scale, int rest, void* workspace, size_t workspace_bytes, void* stream) {
  if (int s = step_dims_status(d)) return s;
  if (!out || !q || !q->p || !kpool || !vpool || !kv || !plan) return PIE_ENULL;
  if ((D != 64 && D != 128) || !(scale > 0.f) || kv->tok_stride <= 0 || kv->tok_stride % 8 || kv->head_stride % 8 || q->stride_h % 8 || q->stride_l % 8)
    return PIE_EINVAL_SHAPE;
  for (const void* p : {(const void*)out, q->p, kpool, vpool, (const void*)plan, (const void*)workspace})
    if (reinterpret_cast<uintptr_t>(p) & 15) return PIE_EALIGN;
  if (!workspace || workspace_bytes < pie_chunk_attn_workspace_bytes(d, D)) return PIE_EWORKSPACE;
  ChunkArgs a;
  a.out = (uint16_t*)out; a.q = (const uint16_t*)q->p; a.k = (const uint16_t*)kpool; a.v = (const uint16_t*)vpool;
  a.q_row = q->stride_l; a.q_head = q->stride_h; a.tok = kv->tok_stride; a.head = kv->head_stride;
  a.plan = plan; a.l = step_layout(*d); a.d = *d; a.scale_log2e = scale * 1.4426950408889634f; a.rest = rest;
  const dim3 grid(d->rows, (d->Hq + 3) / 4);
  count_launch();
  return status_of(D == 128 ? launch_pdl(chunk_attn_kernel<128>, grid, dim3(128), 0, (cudaStream_t)stream, a)
                            : launch_pdl(chunk_attn_kernel<64>, grid, dim3(128), 0, (cudaStream_t)stream, a));
}

}  // extern "C"
