// A ragged step's rows into a cache of 8 bits (include/pie_b200.h): queries rotated, keys rotated and values, as e4m3 with a power of two for a scale for each page and head.
//
// A CTA has a page of one key / value head: the rows of the step that go there, at most 64, are held in registers (keys as they are rotated, in fp32), their largest magnitude
// is taken over the CTA, and each feature is read once and written once.  A scale that grows is a power of two times the one before, so what the page held is brought to it
// without another rounding, but for what falls below e4m3's lowest.  Which page a CTA has is found from the plan: request s may have the places 2 s + row_starts[s] / 64 and up
// to the next one's, which are as many as the pages it writes to, or more (the others' CTAs leave).  Further CTAs rotate the queries, a thread eight pairs of features.
// HBM-bound where there are many rows; where there are few, the chain is row starts, slot, keys and scale, one reduction, codes.
#include "pie_ptx.cuh"
#include "pie_step_plan.h"

namespace pie {

struct Fp8Args {
  uint16_t* q_out;
  uint8_t *kp, *vp;
  float *ks, *vs;
  RopeRows r;
  const int32_t *row_starts, *contexts, *positions, *slots;
  const float* freqs;
  int requests, rows, pages, Hq, Hkv, rest;
  int page_ctas, HL;       // CTAs of pages; threads that share a row's queries / 8 pairs
  int heads;               // of a CTA of pages, one after the other
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) { return e4m3x2(a, b) | (e4m3x2(c, d) << 16); }
// four codes, times f
__device__ __forceinline__ uint32_t e4m3x4_times(uint32_t w, float f) {
  float v[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t x;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(x) : "h"((uint16_t)(w >> (16 * h))));
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(v[2 * h]), "=f"(v[2 * h + 1]) : "r"(x));
  }
  return e4m3x4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
}
// eight pairs of a head: features i and i + D / 2
__device__ __forceinline__ void turn8(const uint4& v1, const uint4& v2, const float (&cs)[8], const float (&sn)[8], float (&o1)[8], float (&o2)[8]) {
  const uint32_t a[4] = {v1.x, v1.y, v1.z, v1.w}, c[4] = {v2.x, v2.y, v2.z, v2.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x1 = e & 1 ? bf16hi(a[e >> 1]) : bf16lo(a[e >> 1]), x2 = e & 1 ? bf16hi(c[e >> 1]) : bf16lo(c[e >> 1]);
    o1[e] = __fsub_rn(__fmul_rn(x1, cs[e]), __fmul_rn(x2, sn[e]));
    o2[e] = __fadd_rn(__fmul_rn(x1, sn[e]), __fmul_rn(x2, cs[e]));
  }
}
__device__ __forceinline__ void angles8(float position, const float* freqs, float (&cs)[8], float (&sn)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) rope_sincos(position * (1.0f / freqs[e]), &sn[e], &cs[e]);
}
// sin / cos of an angle of up to 2^17 to the last place or so (rope_sincos is off by 5e-7, which a rounding to bf16 hides and one to a code, next to a border, shows): the angle less the nearest
// multiple k of pi / 2, taken off in three pieces -- k has 17 bits, so that the first difference is exact --, and Taylor's polynomials on what is left, at most pi / 4 (next terms 2e-9).
__device__ __forceinline__ void sincos_of(float theta, float& sn, float& cs) {
  const float k = rintf(theta * 0.636619772f);
  float r = fmaf(-k, 1.57079637f, theta);
  r = fmaf(-k, -4.37113883e-8f, r);
  r = fmaf(-k, -1.71512451e-15f, r);
  const float z = r * r;
  float s = fmaf(z, fmaf(z, fmaf(z, 2.75573192e-6f, -1.98412698e-4f), 8.33333333e-3f), -0.166666667f);
  s = fmaf(r * z, s, r);
  float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.75573192e-7f, 2.48015873e-5f), -1.38888889e-3f), 4.16666667e-2f), -0.5f);
  c = fmaf(z, c, 1.f);
  const int q = (int)k;
  const float a = q & 1 ? c : s, b = q & 1 ? s : c;
  sn = q & 2 ? -a : a;
  cs = (q + 1) & 2 ? -b : b;
}
// the lowest power of two, 2^-60 at least, with which a magnitude is 448 or less; NaN for what is not finite
__device__ __forceinline__ float e4m3_scale(uint32_t bits) {
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);   // (448 = 1.75 2^8)
  return __uint_as_float((uint32_t)max(e, 127 - 60) << 23);
}

template <int D>
__global__ void __launch_bounds__(256, 3) rope_kv_fp8_kernel(const __grid_constant__ Fp8Args a) {
  constexpr int half = D / 2, PB = half / 8, VC = D / 8;     // pieces of eight: pairs of a head, features of a head
  constexpr int KN = 64 * PB / 256, VN = 64 * VC / 256;      // of a page, a thread
  __shared__ uint32_t most[2][2][8];
  __shared__ float4 angles[KN][4][256];                      // a thread's own: cosines, sines of its pairs
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x >= a.page_ctas) {
    // ------------------------------------------------------------------------------------------------ queries
    const int pb = tid % PB, rem = tid / PB, hl = rem % a.HL, l = ((int)blockIdx.x - a.page_ctas) * (256 / PB / a.HL) + rem / a.HL;
    if (l >= a.rows) return;
    const int slot = __ldg(a.slots + l);
    uint16_t* const qo = a.q_out + (size_t)l * a.Hq * D + pb * 8;
    if (slot < 0 || slot >= a.pages * kStepPage) {
      if (a.rest)
        for (int h = hl; h < a.Hq; h += a.HL)
          *reinterpret_cast<uint4*>(qo + (size_t)h * D) = *reinterpret_cast<uint4*>(qo + (size_t)h * D + half) = make_uint4(0, 0, 0, 0);
      return;
    }
    float sn[8], cs[8];
    angles8((float)__ldg(a.positions + l), a.freqs + pb * 8, cs, sn);
    const uint16_t* const src = a.r.q + l * a.r.qs.sl + pb * 8;
    for (int h0 = hl; h0 < a.Hq; h0 += 4 * a.HL) {   // the loads of four heads in flight before the first store
      uint4 v1[4], v2[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (h0 + i * a.HL < a.Hq) {
          v1[i] = *reinterpret_cast<const uint4*>(src + (h0 + i * a.HL) * a.r.qs.sh);
          v2[i] = *reinterpret_cast<const uint4*>(src + (h0 + i * a.HL) * a.r.qs.sh + half);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (h0 + i * a.HL >= a.Hq) break;
        float o1[8], o2[8];
        turn8(v1[i], v2[i], cs, sn, o1, o2);
        uint16_t* const o = qo + (size_t)(h0 + i * a.HL) * D;
        *reinterpret_cast<uint4*>(o) = make_uint4(pack_bf16(o1[0], o1[1]), pack_bf16(o1[2], o1[3]), pack_bf16(o1[4], o1[5]), pack_bf16(o1[6], o1[7]));
        *reinterpret_cast<uint4*>(o + half) = make_uint4(pack_bf16(o2[0], o2[1]), pack_bf16(o2[2], o2[3]), pack_bf16(o2[4], o2[5]), pack_bf16(o2[6], o2[7]));
      }
    }
    return;
  }
  // -------------------------------------------------------------------------------------------------- a page of a head
  const int sets = (a.Hkv + a.heads - 1) / a.heads, head0 = (int)blockIdx.x % sets * a.heads, place = (int)blockIdx.x / sets;
  // the last request whose places begin at or below this one: every so many-th of them, then those between
  int s = 0, n_rows = 0, row0 = 0;
  for (int stride = (a.requests + 255) / 256, span = a.requests;; span = stride, stride = 1) {
    const int at = s + tid * stride;
    const bool below = tid * stride < span && at < a.requests && 2 * at + __ldg(a.row_starts + at) / kStepPage <= place;
    s += (__syncthreads_count(below) - 1) * stride;   // (request 0's begin at 0)
    if (stride == 1) break;
  }
  row0 = __ldg(a.row_starts + s);
  n_rows = __ldg(a.row_starts + s + 1) - row0;
  const int context = __ldg(a.contexts + s), j = place - (2 * s + row0 / kStepPage), page = context / kStepPage + j;
  const int lies = j == 0 ? context % kStepPage : 0, skipped = j == 0 ? 0 : page * kStepPage - context;   // tokens that the page holds; rows that go to pages before it
  const int count = min(kStepPage - lies, n_rows - skipped);
  if (count <= 0) return;
  row0 += skipped;
  const int slot = __ldg(a.slots + row0);
  if (slot < 0 || slot >= a.pages * kStepPage) return;
  {
    float inv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) inv[e] = 1.0f / __ldg(a.freqs + tid % PB * 8 + e);
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const int t = (tid + 256 * i) / PB;
      if (t >= count) break;
      float sn[8], cs[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) sincos_of((float)(page * kStepPage + lies + t) * inv[e], sn[e], cs[e]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        angles[i][h][tid] = make_float4(cs[4 * h], cs[4 * h + 1], cs[4 * h + 2], cs[4 * h + 3]);
        angles[i][2 + h][tid] = make_float4(sn[4 * h], sn[4 * h + 1], sn[4 * h + 2], sn[4 * h + 3]);
      }
    }
  }
  auto turned = [&](int i, const uint4& k1, const uint4& k2, float (&o1)[8], float (&o2)[8]) {
    float cs[8], sn[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<float4*>(cs + 4 * h) = angles[i][h][tid];
      *reinterpret_cast<float4*>(sn + 4 * h) = angles[i][2 + h][tid];
    }
    turn8(k1, k2, cs, sn, o1, o2);
  };
#pragma unroll 1
  for (int head = head0; head < min(head0 + a.heads, a.Hkv); ++head) {
    const size_t block = (size_t)(slot / kStepPage) * a.Hkv + head;
    uint8_t* const kp = a.kp + block * kStepPage * D;
    uint8_t* const vp = a.vp + block * kStepPage * D;
    const float had_k = lies ? a.ks[block] : 0.f, had_v = lies ? a.vs[block] : 0.f;

    uint4 v[VN], k1[KN], k2[KN];
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const int t = (tid + 256 * i) / PB, pb = tid % PB;
      k1[i] = k2[i] = make_uint4(0, 0, 0, 0);
      if (t < count) {
        const uint16_t* const src = a.r.k + (row0 + t) * a.r.ks.sl + head * a.r.ks.sh + pb * 8;
        k1[i] = *reinterpret_cast<const uint4*>(src);
        k2[i] = *reinterpret_cast<const uint4*>(src + half);
      }
    }
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const int t = (tid + 256 * i) / VC, c = tid % VC;
      v[i] = make_uint4(0, 0, 0, 0);
      if (t < count) v[i] = *reinterpret_cast<const uint4*>(a.r.v + (row0 + t) * a.r.vs.sl + head * a.r.vs.sh + c * 8);
    }
    uint32_t mk = 0, mv = 0;   // magnitudes in the order of their bits
#pragma unroll
    for (int i = 0; i < KN; ++i)
      if ((tid + 256 * i) / PB < count) {
        float o1[8], o2[8];
        turned(i, k1[i], k2[i], o1, o2);
#pragma unroll
        for (int e = 0; e < 8; ++e) mk = max(mk, max(__float_as_uint(o1[e]) & 0x7fffffffu, __float_as_uint(o2[e]) & 0x7fffffffu));
      }
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      constexpr uint32_t ABS = 0x7fff7fffu;
      const uint32_t m = __vmaxu2(__vmaxu2(v[i].x & ABS, v[i].y & ABS), __vmaxu2(v[i].z & ABS, v[i].w & ABS));
      mv = max(mv, max(m << 16, m & 0xffff0000u));
    }
    mk = __reduce_max_sync(0xffffffffu, mk);
    mv = __reduce_max_sync(0xffffffffu, mv);
    if (lane == 0) { most[head & 1][0][warp] = mk; most[head & 1][1][warp] = mv; }   // (two of them: a warp may be at the next head)
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) { mk = max(mk, most[head & 1][0][w]); mv = max(mv, most[head & 1][1][w]); }
    const float need_k = e4m3_scale(mk), need_v = e4m3_scale(mv);
    const float sk = had_k >= need_k || had_k != had_k ? had_k : need_k, sv = had_v >= need_v || had_v != had_v ? had_v : need_v;
    const float ik = 1.f / sk, iv = 1.f / sv;
    if (tid == 0) { a.ks[block] = sk; a.vs[block] = sv; }   // (every thread's had_k, had_v lie behind the barrier's other side)
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const int t = (tid + 256 * i) / PB, pb = tid % PB;
      if (t < count) {
        float o1[8], o2[8];   // (once more: sooner done than held)
        turned(i, k1[i], k2[i], o1, o2);
        uint8_t* const to = kp + (lies + t) * D + pb * 8;
        *reinterpret_cast<uint2*>(to) = make_uint2(e4m3x4(o1[0] * ik, o1[1] * ik, o1[2] * ik, o1[3] * ik), e4m3x4(o1[4] * ik, o1[5] * ik, o1[6] * ik, o1[7] * ik));
        *reinterpret_cast<uint2*>(to + half) = make_uint2(e4m3x4(o2[0] * ik, o2[1] * ik, o2[2] * ik, o2[3] * ik), e4m3x4(o2[4] * ik, o2[5] * ik, o2[6] * ik, o2[7] * ik));
      }
    }
#pragma unroll
    for (int i = 0; i < VN; ++i) {
      const int t = (tid + 256 * i) / VC, c = tid % VC;
      if (t < count)
        *reinterpret_cast<uint2*>(vp + (lies + t) * D + c * 8) =
            make_uint2(e4m3x4(bf16lo(v[i].x) * iv, bf16hi(v[i].x) * iv, bf16lo(v[i].y) * iv, bf16hi(v[i].y) * iv),
                       e4m3x4(bf16lo(v[i].z) * iv, bf16hi(v[i].z) * iv, bf16lo(v[i].w) * iv, bf16hi(v[i].w) * iv));
    }
    // what the page held, where its scale has grown
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const float had = kv ? had_v : had_k, now = kv ? sv : sk;
      if (!(now > had)) continue;
      const float f = had / now;
      uint4* const p = reinterpret_cast<uint4*>(kv ? vp : kp);
      for (int i = tid; i < lies * (D / 16); i += 256) {
        const uint4 w = p[i];
        p[i] = make_uint4(e4m3x4_times(w.x, f), e4m3x4_times(w.y, f), e4m3x4_times(w.z, f), e4m3x4_times(w.w, f));
      }
    }
  }
}

}  // namespace pie

using namespace pie;

extern "C" int pie_rope_kv_fp8(void* q_out, uint8_t* kpool, float* k_scales, uint8_t* vpool, float* v_scales, const pie_head_rows* q, const pie_head_rows* k,
                               const pie_head_rows* v, const int32_t* plan, const pie_step_dims* d, const float* freqs, int D, int rest, void* stream) {
  if (int s = step_dims_status(d)) return s;
  if (!q_out || !kpool || !k_scales || !vpool || !v_scales || !q || !k || !v || !q->p || !k->p || !v->p || !plan || !freqs) return PIE_ENULL;
  if (D != 64 && D != 128) return PIE_EINVAL_SHAPE;
  const StepLayout l = step_layout(*d);
  Fp8Args a;
  const pie_head_rows* src[3] = {q, k, v};
  const uint16_t** at[3] = {&a.r.q, &a.r.k, &a.r.v};
  KvSrc* st[3] = {&a.r.qs, &a.r.ks, &a.r.vs};
  for (int i = 0; i < 3; ++i) {
    if (src[i]->stride_h % 8 || src[i]->stride_l % 8) return PIE_EINVAL_SHAPE;
    *at[i] = (const uint16_t*)src[i]->p;
    *st[i] = {0, src[i]->stride_h, src[i]->stride_l};
  }
  for (const void* p : {(const void*)q_out, (const void*)kpool, (const void*)vpool, q->p, k->p, v->p, (const void*)plan})
    if (reinterpret_cast<uintptr_t>(p) & 15) return PIE_EALIGN;
  a.q_out = (uint16_t*)q_out; a.kp = kpool; a.vp = vpool; a.ks = k_scales; a.vs = v_scales;
  a.row_starts = plan + l.row_starts; a.contexts = plan + l.contexts; a.positions = plan + l.positions; a.slots = plan + l.slots;
  a.freqs = freqs;
  a.requests = d->requests; a.rows = d->rows; a.pages = d->pages; a.Hq = d->Hq; a.Hkv = d->Hkv; a.rest = rest;
  const int lanes = 256 / (D / 16);
  a.HL = d->rows >= 1024 ? 4 : lanes;
  const int per = lanes / a.HL;
  // Heads that share a row's angles, as many as leave each SM a CTA of full pages (8191 rows of 8 heads: one a CTA 42.7 us, two 42.4, four 37.1).
  const long long blocks = d->rows / kStepPage * (long long)d->Hkv;
  a.heads = blocks >= 4LL * num_sms() ? 4 : blocks >= 2LL * num_sms() ? 2 : 1;
  const long long pages = (2LL * d->requests + d->rows / kStepPage) * ((d->Hkv + a.heads - 1) / a.heads), grid = pages + (d->rows + per - 1) / per;
  if (grid > 0x7fffffff) return PIE_EINVAL_SHAPE;
  a.page_ctas = (int)pages;
  count_launch();
  return status_of(D == 128 ? launch_pdl(rope_kv_fp8_kernel<128>, dim3((unsigned)grid), dim3(256), 0, (cudaStream_t)stream, a)
                            : launch_pdl(rope_kv_fp8_kernel<64>, dim3((unsigned)grid), dim3(256), 0, (cudaStream_t)stream, a));
}
