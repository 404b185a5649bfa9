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
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "kv_page.cuh"
#include "lk_api.h"

namespace lk {

// ---------------------------------------------------------------- append
// A run is the rows of a call that go to one page: consecutive rows with
// consecutive slots.  One warp takes a run's keys or values of one head: 16 bytes
// (8 dims) a lane, RPI rows at a time, the first 8 of those steps kept in registers
// between the pass for the maximum and the pass that encodes, which is all of a page
// of 16 rows (32 at head_dim 64); longer runs read the rest again, from L1 or L2.
//
// Bound by HBM for a prompt (6 bytes a value with the codes written: 8190 rows of 8
// heads x 128 in 9 to 12 us), by the chain slot -> row -> maximum -> store for a token
// per sequence (256 rows 4.1 us).  A block's warps look for runs that start in its `window`
// rows and take them one after another: few rows want a block per run, prompts few blocks
// without one (15 of 16 rows start none).  Windows of 1 / 4 / 16 rows, us: 256 sequences'
// tokens 4.1 / 6.2 / 20, 1000 of them 10.2 / 10.8 / 20; 1000 rows of a prompt 5.9 / 4.6 / 4.6,
// 4000 13.7 / 8.0 / 6.2, 8190 25 / 12.7 / 9.0.

// 8 bf16 -> 8 codes.  CHECK: some of them are not finite (infinities saturate, NaN -> 0).
template <int KV, bool CHECK>
__device__ __forceinline__ uint2 encode8(uint4 x, float inv) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t out[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = unpack_bf16x2(w[i]);
    f.x *= inv, f.y *= inv;
    uint32_t two;
    if constexpr (CHECK) two = page_encode<KV>(f.x) | page_encode<KV>(f.y) << 8;
    else if constexpr (KV == 1) two = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
    else two = (__float2int_rn(f.x) & 0xFF) | (__float2int_rn(f.y) & 0xFF) << 8;
    out[i / 2] |= two << (16 * (i & 1));
  }
  return make_uint2(out[0], out[1]);
}

// 8 codes moved to a larger scale (f = old / new <= 1): always finite.
template <int KV>
__device__ __forceinline__ uint2 move8(uint2 c, float f) {
  uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t out = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) out |= (uint32_t)page_encode<KV>(page_decode<KV>((uint8_t)(w[i] >> (8 * k))) * f) << (8 * k);
    w[i] = out;
  }
  return make_uint2(w[0], w[1]);
}

// largest |x| bits of 8 bf16, as the larger of two 16-bit halves
__device__ __forceinline__ uint32_t top8(uint32_t top, uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) top = __vmaxu2(top, w[i] & 0x7FFF7FFFu);
  return top;
}

template <int KV, int DH>
__device__ void append_run(const LkPageAppendDesc& d, int t, int rows, int slot, int h, bool value) {
  constexpr int LPR = DH / 8, RPI = 32 / LPR, HELD = 8;
  const int lane = threadIdx.x & 31, sub = lane / LPR, col = lane % LPR * 8;
  const int64_t pg = slot / d.page;
  const int first = slot - (int)pg * d.page;
  const __nv_bfloat16* src =
      (const __nv_bfloat16*)d.qkv + (int64_t)t * d.ld + (d.Hq + (value ? d.Hkv : 0) + h) * DH + col;
  const int64_t pitch = (int64_t)d.Hkv * DH;
  uint8_t* dst = (uint8_t*)(value ? d.v_cache : d.k_cache) + slot * pitch + h * DH + col;
  float* scale = (value ? d.v_scale : d.k_scale) + pg * d.Hkv + h;
  const float old = first > 0 ? *scale : 0.f;
  uint4 x[HELD];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int r = i * RPI + sub;
    x[i] = make_uint4(0, 0, 0, 0);
    if (r < rows) x[i] = *reinterpret_cast<const uint4*>(src + r * d.ld);
  }
#pragma unroll
  for (int i = 0; i < HELD; ++i) top = top8(top, x[i]);
  for (int r = HELD * RPI + sub; r < rows; r += RPI) top = top8(top, *reinterpret_cast<const uint4*>(src + r * d.ld));
  top = max(top & 0xFFFFu, top >> 16);
  const bool special = __any_sync(0xffffffffu, top >= 0x7F80u);  // infinities or NaN among them
  if (special) {  // the maximum of the finite ones
    top = 0;
    for (int r = sub; r < rows; r += RPI)
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = __bfloat16_as_ushort(src[r * d.ld + i]) & 0x7FFFu;
        if (a < 0x7F80u) top = max(top, a);
      }
  }
  float now = page_scale<KV>(__uint_as_float(__reduce_max_sync(0xffffffffu, top) << 16));
  if (first > 0 && old >= now) now = old;
  else if (first > 0) {  // the rows already there move to the new scale
    const float f = old / now;
    for (int r = sub; r < first; r += RPI) {
      uint2* c = reinterpret_cast<uint2*>(dst + (r - first) * pitch);
      *c = move8<KV>(*c, f);
    }
  }
  const float inv = 1.f / now;
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int r = i * RPI + sub;
    if (r < rows) *reinterpret_cast<uint2*>(dst + r * pitch) = special ? encode8<KV, true>(x[i], inv) : encode8<KV, false>(x[i], inv);
  }
  for (int r = HELD * RPI + sub; r < rows; r += RPI) {
    const uint4 y = *reinterpret_cast<const uint4*>(src + r * d.ld);
    *reinterpret_cast<uint2*>(dst + r * pitch) = special ? encode8<KV, true>(y, inv) : encode8<KV, false>(y, inv);
  }
  if (lane == 0) *scale = now;
}

// grid (windows of rows, groups of 8 (head, K|V) pairs)
template <int KV, int DH>
__global__ void __launch_bounds__(256, 4) page_append_kernel(LkPageAppendDesc d, int window) {
  const int item = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= 2 * d.Hkv) return;
  // lane l looks at row t0 - 1 + l: which rows continue the row before them
  const int t0 = blockIdx.x * window, t = t0 - 1 + lane;
  const int s = t >= 0 && t < d.T ? d.slots[t] : -1;
  const int before = __shfl_up_sync(0xffffffffu, s, 1);
  const bool more = lane > 0 && s > 0 && before >= 0 && s == before + 1 && s % d.page != 0;
  const unsigned goes_on = __ballot_sync(0xffffffffu, more);
  unsigned starts = __ballot_sync(0xffffffffu, lane > 0 && lane <= window && s >= 0 && !more);
  while (starts) {
    const int l = __ffs(starts) - 1;
    starts &= starts - 1;
    const int slot = __shfl_sync(0xffffffffu, s, l);
    if (slot >= d.num_slots) {
      if (lane == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
      continue;
    }
    const unsigned rest = l == 31 ? 0u : goes_on >> (l + 1);
    int rows = 1 + __ffs(~rest) - 1;  // rest has a zero: its top bit
    if (l + rows == 32) {             // as far as this warp looked: on from there
      const int room = d.page - slot % d.page;
      for (bool all = true; all;) {
        const int tr = t0 - 1 + l + rows + lane;
        const bool here = rows + lane < room && tr < d.T && d.slots[tr] == slot + rows + lane;
        const unsigned m = __ballot_sync(0xffffffffu, here);
        all = m == 0xffffffffu;
        rows += all ? 32 : __ffs(~m) - 1;
      }
    }
    append_run<KV, DH>(d, t0 - 1 + l, rows, slot, item >> 1, item & 1);
  }
}

// ---------------------------------------------------------------- gather
// A thread takes 8 codes of a token's keys and the same 8 of its values (the heads of a
// slot lie side by side in the cache and in the output alike): two 8-byte loads, two
// 16-byte stores, a warp's stores in one piece.  Bound by HBM: 3 bytes a value.
template <int KV>
__device__ __forceinline__ uint4 widen8(uint2 c, float scale) {
  const uint32_t w[2] = {c.x, c.y};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    const uint32_t two = w[i / 2] >> (16 * (i & 1));
    if constexpr (KV == 1) {
      const __half2_raw h2 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(two & 0xFFFFu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
      a = f.x, b = f.y;
    } else {
      a = (float)(int8_t)(two & 0xFFu), b = (float)(int8_t)(two >> 8 & 0xFFu);
    }
    o[i] = pack_bf16x2(a * scale, b * scale);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int KV>
__global__ void __launch_bounds__(256) page_gather_kernel(LkPageGatherDesc d, int total, FastDiv per_row, FastDiv page) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int t = per_row.div(i), at = (i - t * per_row.d) * 8;
  const int h = at >> (d.Dh == 64 ? 6 : 7), width = d.Hkv * d.Dh;
  const int slot = d.slots[t];
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (slot < 0 || slot >= d.num_slots) {
    if (d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
  } else {
    const int64_t sc = (int64_t)page.div(slot) * d.Hkv + h, from = (int64_t)slot * width + at;
    const uint2 kc = *reinterpret_cast<const uint2*>((const uint8_t*)d.k_cache + from);
    const uint2 vc = *reinterpret_cast<const uint2*>((const uint8_t*)d.v_cache + from);
    k = widen8<KV>(kc, d.k_scale[sc]);
    v = widen8<KV>(vc, d.v_scale[sc]);
  }
  __nv_bfloat16* out = (__nv_bfloat16*)d.out + (int64_t)t * d.ldo + at;
  *reinterpret_cast<uint4*>(out) = k;
  *reinterpret_cast<uint4*>(out + width) = v;
}

// ---------------------------------------------------------------- page copies
// grid (items, tensors), an item being a chunk of a page (fastest), a layer, a move: PER threads copy PER * 64 bytes of one page
// of one layer of one tensor, every load on its way before the first store: a block 8 KB, or
// a warp 2 KB where pages are no larger (one block each took 47 us for 41600 pages of 256
// bytes, a warp each 20).  Bound by HBM (1500 pages of 8 KB in 22 layers of two tensors: 169
// us, 98 % of the copy rate).
constexpr int COPY_THREADS = 128, COPY_AHEAD = 4;

template <int PER, typename T>
__device__ __forceinline__ void copy_as(const char* src, char* dst, int bytes) {
  const int n = bytes / (int)sizeof(T);
  for (int i = threadIdx.x % PER; i < n; i += COPY_AHEAD * PER) {
    T x[COPY_AHEAD];
#pragma unroll
    for (int k = 0; k < COPY_AHEAD; ++k)
      if (i + k * PER < n) x[k] = ((const T*)src)[i + k * PER];
#pragma unroll
    for (int k = 0; k < COPY_AHEAD; ++k)
      if (i + k * PER < n) ((T*)dst)[i + k * PER] = x[k];
  }
}

template <int PER>
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(LkCopyPagesDesc d, int total, FastDiv chunks, FastDiv layers) {
  const int item = blockIdx.x * (COPY_THREADS / PER) + threadIdx.x / PER;
  if (item >= total) return;
  const int a = chunks.div(item), m = layers.div(a), layer = a - m * d.layers;
  const int64_t bytes = d.page_bytes[blockIdx.y], from = (int64_t)(item - a * chunks.d) * (PER * COPY_AHEAD * 16);
  const int src = d.moves[2 * m], dst = d.moves[2 * m + 1];
  if (src < 0 || dst < 0 || src >= d.num_pages || dst >= d.num_pages) {
    if (threadIdx.x % PER == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    return;
  }
  if (from >= bytes) return;
  char* base = (char*)d.base[blockIdx.y] + (int64_t)layer * d.num_pages * bytes + from;
  const char* s = base + src * bytes;
  char* t = base + dst * bytes;
  const int n = (int)min(bytes - from, (int64_t)(PER * COPY_AHEAD * 16));
  if (((uintptr_t)s | (uintptr_t)t | (uintptr_t)n) % 16 == 0) copy_as<PER, uint4>(s, t, n);
  else if (((uintptr_t)s | (uintptr_t)t | (uintptr_t)n) % 4 == 0) copy_as<PER, uint32_t>(s, t, n);
  else copy_as<PER, uint8_t>(s, t, n);
}

}  // namespace lk

using namespace lk;

extern "C" int lk_page_append(const LkPageAppendDesc* d, cudaStream_t s) {
  LK_REQUIRE(d->Dh == 64 || d->Dh == 128, "page_append: head_dim must be 64 or 128");
  if (d->T == 0 || d->Hkv == 0) return 0;
  LK_REQUIRE(d->Hkv <= 4 * 65535, "page_append: too many heads");
  const int window = d->T <= 512 ? 1 : d->T <= 2048 ? 4 : 16;
  const dim3 grid(cdiv(d->T, window), cdiv(2 * d->Hkv, 8));
  if (d->kv_dtype == 1)
    d->Dh == 64 ? page_append_kernel<1, 64><<<grid, 256, 0, s>>>(*d, window) : page_append_kernel<1, 128><<<grid, 256, 0, s>>>(*d, window);
  else
    d->Dh == 64 ? page_append_kernel<2, 64><<<grid, 256, 0, s>>>(*d, window) : page_append_kernel<2, 128><<<grid, 256, 0, s>>>(*d, window);
  return check_launch("page_append");
}

extern "C" int lk_page_gather(const LkPageGatherDesc* d, cudaStream_t s) {
  const int per_row = d->Hkv * d->Dh / 8;
  const int64_t total = (int64_t)d->n * per_row;
  if (total == 0) return 0;
  LK_REQUIRE(total <= (1ll << 31) - 256, "page_gather: too many rows in one call");  // the last block's items are ints too
  const int grid = cdiv(total, 256);
  if (d->kv_dtype == 1)
    page_gather_kernel<1><<<grid, 256, 0, s>>>(*d, (int)total, FastDiv(per_row), FastDiv(d->page));
  else
    page_gather_kernel<2><<<grid, 256, 0, s>>>(*d, (int)total, FastDiv(per_row), FastDiv(d->page));
  return check_launch("page_gather");
}

extern "C" int lk_copy_pages(const LkCopyPagesDesc* d, cudaStream_t s) {
  if (d->num_moves == 0 || d->layers == 0 || d->tensors == 0) return 0;
  int64_t most = 1;
  for (int i = 0; i < d->tensors; ++i) most = std::max(most, d->page_bytes[i]);
  const int per = most <= 32 * COPY_AHEAD * 16 ? 32 : COPY_THREADS, share = per * COPY_AHEAD * 16;
  const int64_t chunks = (most + share - 1) / share, total = (int64_t)d->num_moves * d->layers * chunks;
  LK_REQUIRE(total < (1ll << 31) - COPY_THREADS, "copy_pages: too many moves in one call");
  const dim3 grid(cdiv(total * per, COPY_THREADS), d->tensors);
  const FastDiv c((int)chunks), l(d->layers);
  per == 32 ? copy_pages_kernel<32><<<grid, COPY_THREADS, 0, s>>>(*d, (int)total, c, l)
            : copy_pages_kernel<COPY_THREADS><<<grid, COPY_THREADS, 0, s>>>(*d, (int)total, c, l);
  return check_launch("copy_pages");
}
