// Attention of the newest q_len tokens of each sequence over the page-scaled
// 8-bit KV cache (csrc/kv_page.cu describes the cache).
//
//   s[t] = (q . k[t]) * scale * kscale[page(t)],  t <= position of the query
//   out  = sum_t softmax(s)[t] * v[t] * vscale[page(t)]
//
// Query j of a sequence of ctx tokens sits at position ctx - q_len + j.  A query
// without a token before it (an unused batch row of ctx 0) gives zeros.
#include "common.cuh"
#include "host_util.h"
#include "kv_page.cuh"
#include "lk_api.h"

namespace lk {

// One block per (query row, query head); each warp takes every fourth token
// with its lanes over the head dimension, and the four running softmaxes are
// merged at the end.
template <int KV, int DH>
__global__ void __launch_bounds__(128) page_attn_kernel(LkPageAttnDesc d) {
  constexpr int PER = DH / 32;
  __shared__ float sm_m[4], sm_l[4], sm_o[4][DH];
  const int row = blockIdx.x, head = blockIdx.y;
  const int seq = row / d.q_len, h = head / (d.Hq / d.Hkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int ctx = d.ctx_lens[seq];
  if (ctx > (int64_t)d.max_pages * d.page) {
    if (threadIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    ctx = d.max_pages * d.page;
  }
  const int upto = ctx - d.q_len + row % d.q_len + 1;
  const int* table = d.tables + (int64_t)seq * d.max_pages;
  const __nv_bfloat16* q = (const __nv_bfloat16*)d.q + (int64_t)row * d.ldq + head * DH;
  float qf[PER], o[PER], m = -INFINITY, l = 0.f;
  for (int i = 0; i < PER; ++i) {
    qf[i] = __bfloat162float(q[i * 32 + lane]);
    o[i] = 0.f;
  }
  const float sl2 = d.scale * 1.4426950408889634f;
  for (int t = warp; t < upto; t += 4) {
    const int pg = table[t / d.page];
    if (pg < 0 || pg >= d.num_pages) {
      if (lane == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
      continue;
    }
    const int64_t at = (((int64_t)pg * d.page + t % d.page) * d.Hkv + h) * DH + lane;
    float s = 0.f;
    for (int i = 0; i < PER; ++i) s += qf[i] * page_decode<KV>(((const uint8_t*)d.k_cache)[at + i * 32]);
    s = warp_sum(s) * sl2 * d.k_scale[(int64_t)pg * d.Hkv + h];
    const float mn = fmaxf(m, s);
    const float a = m == -INFINITY ? 0.f : exp2f(m - mn), p = exp2f(s - mn);
    m = mn;
    l = l * a + p;
    const float pv = p * d.v_scale[(int64_t)pg * d.Hkv + h];
    for (int i = 0; i < PER; ++i) o[i] = o[i] * a + pv * page_decode<KV>(((const uint8_t*)d.v_cache)[at + i * 32]);
  }
  if (lane == 0) {
    sm_m[warp] = m;
    sm_l[warp] = l;
  }
  for (int i = 0; i < PER; ++i) sm_o[warp][i * 32 + lane] = o[i];
  __syncthreads();
  for (int c = threadIdx.x; c < DH; c += 128) {
    float M = -INFINITY, L = 0.f, O = 0.f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w]);
    for (int w = 0; w < 4; ++w) {
      const float f = sm_m[w] == -INFINITY ? 0.f : exp2f(sm_m[w] - M);
      L += sm_l[w] * f;
      O += sm_o[w][c] * f;
    }
    ((__nv_bfloat16*)d.out)[(int64_t)row * d.ldo + head * DH + c] = __float2bfloat16(L == 0.f ? 0.f : O / L);
  }
}

}  // namespace lk

using namespace lk;

extern "C" int lk_page_attention(const LkPageAttnDesc* d, cudaStream_t s) {
  LK_REQUIRE(d->Dh == 64 || d->Dh == 128, "page_attention: head_dim must be 64 or 128");
  const int rows = d->num_seqs * d->q_len;
  if (rows == 0) return 0;
  const dim3 grid(rows, d->Hq);
  if (d->kv_dtype == 1)
    d->Dh == 64 ? page_attn_kernel<1, 64><<<grid, 128, 0, s>>>(*d) : page_attn_kernel<1, 128><<<grid, 128, 0, s>>>(*d);
  else
    d->Dh == 64 ? page_attn_kernel<2, 64><<<grid, 128, 0, s>>>(*d) : page_attn_kernel<2, 128><<<grid, 128, 0, s>>>(*d);
  return check_launch("page_attention");
}
