// Page-scaled 8-bit KV cache: append, read-back and page copies.
//
// Cache layout per layer: K and V codes [num_pages * page, Hkv, Dh] (e4m3 or
// int8) and one fp32 scale per (page, KV head), K and V apart, instead of one
// per (token, head): an attention step then reads 8 bytes of scales per page
// and head, and the scale is uniform over the page's rows.
//
// The scale of a page is the power of two 2^e with the smallest e >= -126 such
// that amax <= QMAX 2^e (QMAX 448 or 127; amax over the page's finite values).
// A power of two makes every product with a scale exact, and raising a page's
// scale when a larger token arrives shifts the exponents of the e4m3 codes
// already there: those above the subnormal range keep their values to the bit,
// so a page filled one token at a time holds what one filled at once holds
// (int8 codes lose a bit per doubling).  The cost is up to one bit of the
// code's range, none of an e4m3 normal's precision.
#include "common.cuh"
#include "host_util.h"
#include "kv_page.cuh"
#include "lk_api.h"

namespace lk {

// ---------------------------------------------------------------- append
// Row t starts a run when it does not continue row t - 1 inside one page.
__device__ __forceinline__ bool starts_run(const int* slots, int t, int page) {
  const int s = slots[t];
  return t == 0 || slots[t - 1] < 0 || s != slots[t - 1] + 1 || s % page == 0;
}

// One warp per (row, KV head, K|V); the warps of rows that start a run (the new
// rows of one page) do the run's work: amax, the page's new scale, the codes
// already in the page moved to it when it grew, the new codes.
template <int KV, int DH>
__global__ void page_append_kernel(LkPageAppendDesc d) {
  constexpr int PER = DH / 32;
  const int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= (int64_t)d.T * d.Hkv * 2) return;
  const int which = (int)(w & 1);
  const int h = (int)((w >> 1) % d.Hkv);
  const int t = (int)((w >> 1) / d.Hkv);
  const int slot = d.slots[t];
  if (slot < 0 || !starts_run(d.slots, t, d.page)) return;
  if (slot >= d.num_slots) {
    if (lane == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    return;
  }
  const int pg = slot / d.page, first = slot % d.page;
  int rows = 1;
  while (t + rows < d.T && first + rows < d.page && d.slots[t + rows] == slot + rows) ++rows;
  const __nv_bfloat16* src = (const __nv_bfloat16*)d.qkv + (int64_t)t * d.ld + (d.Hq + which * d.Hkv + h) * DH;
  uint8_t* codes = (uint8_t*)(which ? d.v_cache : d.k_cache);
  float* scale = (which ? d.v_scale : d.k_scale) + (int64_t)pg * d.Hkv + h;
  float amax = 0.f;
  for (int r = 0; r < rows; ++r)
    for (int i = 0; i < PER; ++i) {
      const float a = fabsf(__bfloat162float(src[r * d.ld + i * 32 + lane]));
      if (a <= 3.4028234e38f) amax = fmaxf(amax, a);  // neither inf nor NaN
    }
  float now = page_scale<KV>(warp_max(amax));
  if (first > 0) {
    const float old = *scale;
    now = fmaxf(now, old);
    if (now > old) {
      const float f = old / now;
      for (int r = 0; r < first; ++r)
        for (int i = 0; i < PER; ++i) {
          uint8_t* c = codes + ((int64_t)(pg * (int64_t)d.page + r) * d.Hkv + h) * DH + i * 32 + lane;
          *c = page_encode<KV>(page_decode<KV>(*c) * f);
        }
    }
  }
  const float inv = 1.f / now;
  for (int r = 0; r < rows; ++r)
    for (int i = 0; i < PER; ++i)
      codes[((int64_t)(slot + r) * d.Hkv + h) * DH + i * 32 + lane] =
          page_encode<KV>(__bfloat162float(src[r * d.ld + i * 32 + lane]) * inv);
  __syncwarp();
  if (lane == 0) *scale = now;
}

// ---------------------------------------------------------------- gather
template <int KV>
__global__ void page_gather_kernel(LkPageGatherDesc d) {
  const int64_t total = (int64_t)d.n * 2 * d.Hkv * d.Dh;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int c = (int)(i % d.Dh);
    const int64_t r = i / d.Dh;
    const int h = (int)(r % d.Hkv), which = (int)((r / d.Hkv) & 1), t = (int)(r / (2 * d.Hkv));
    const int slot = d.slots[t];
    float v = 0.f;
    if (slot < 0 || slot >= d.num_slots) {
      if (d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    } else {
      const uint8_t* codes = (const uint8_t*)(which ? d.v_cache : d.k_cache);
      v = page_decode<KV>(codes[((int64_t)slot * d.Hkv + h) * d.Dh + c]) *
          (which ? d.v_scale : d.k_scale)[(int64_t)(slot / d.page) * d.Hkv + h];
    }
    ((__nv_bfloat16*)d.out)[(int64_t)t * d.ldo + (which * d.Hkv + h) * d.Dh + c] = __float2bfloat16(v);
  }
}

// ---------------------------------------------------------------- page copies
// grid (moves * layers, tensors): a block copies one page of one layer of one
// tensor.
template <typename T>
__device__ __forceinline__ void copy_as(const char* src, char* dst, int64_t bytes) {
  for (int64_t i = threadIdx.x; i < bytes / (int64_t)sizeof(T); i += blockDim.x) ((T*)dst)[i] = ((const T*)src)[i];
}

__global__ void copy_pages_kernel(LkCopyPagesDesc d) {
  const int m = blockIdx.x / d.layers, layer = blockIdx.x % d.layers;
  const int src = d.moves[2 * m], dst = d.moves[2 * m + 1];
  if (src < 0 || dst < 0 || src >= d.num_pages || dst >= d.num_pages) {
    if (threadIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    return;
  }
  const int64_t bytes = d.page_bytes[blockIdx.y];
  char* base = (char*)d.base[blockIdx.y] + (int64_t)layer * d.num_pages * bytes;
  const char* a = base + src * bytes;
  char* b = base + dst * bytes;
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)bytes) % 16 == 0) copy_as<uint4>(a, b, bytes);
  else if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)bytes) % 4 == 0) copy_as<uint32_t>(a, b, bytes);
  else copy_as<uint8_t>(a, b, bytes);
}

}  // namespace lk

using namespace lk;

extern "C" int lk_page_append(const LkPageAppendDesc* d, cudaStream_t s) {
  LK_REQUIRE(d->Dh == 64 || d->Dh == 128, "page_append: head_dim must be 64 or 128");
  const int64_t warps = (int64_t)d->T * d->Hkv * 2;
  if (warps == 0) return 0;
  const int grid = cdiv(warps * 32, 256);
  if (d->kv_dtype == 1)
    d->Dh == 64 ? page_append_kernel<1, 64><<<grid, 256, 0, s>>>(*d) : page_append_kernel<1, 128><<<grid, 256, 0, s>>>(*d);
  else
    d->Dh == 64 ? page_append_kernel<2, 64><<<grid, 256, 0, s>>>(*d) : page_append_kernel<2, 128><<<grid, 256, 0, s>>>(*d);
  return check_launch("page_append");
}

extern "C" int lk_page_gather(const LkPageGatherDesc* d, cudaStream_t s) {
  const int64_t work = (int64_t)d->n * 2 * d->Hkv * d->Dh;
  if (work == 0) return 0;
  const int grid = (int)std::min<int64_t>((work + 255) / 256, (int64_t)num_sms() * 8);
  d->kv_dtype == 1 ? page_gather_kernel<1><<<grid, 256, 0, s>>>(*d) : page_gather_kernel<2><<<grid, 256, 0, s>>>(*d);
  return check_launch("page_gather");
}

extern "C" int lk_copy_pages(const LkCopyPagesDesc* d, cudaStream_t s) {
  if (d->num_moves == 0 || d->layers == 0 || d->tensors == 0) return 0;
  LK_REQUIRE((int64_t)d->num_moves * d->layers < (1ll << 31), "copy_pages: too many moves in one call");
  copy_pages_kernel<<<dim3(d->num_moves * d->layers, d->tensors), 256, 0, s>>>(*d);
  return check_launch("copy_pages");
}
