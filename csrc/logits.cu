// Logits before sampling: penalties for tokens already seen, biases and
// grammar masks, and the token counts that the penalties read.
//
//   counts [rows, V] int16: bit 15 = the token is in the prompt, bits 0-14 = how
//   often it was generated (saturating at 32767)
//   z > 0 ? z / r : z * r   for tokens seen (repetition penalty r)
//   z - f * count - p * [count > 0]    (frequency f, presence p)
//   z + bias;  -inf where the row's grammar does not allow the token
// in fp32 from the logits' type and rounded to it once.
#include "common.cuh"
#include "host_util.h"
#include "lk_api.h"

namespace lk {

constexpr int ADJ_THREADS = 256;
constexpr int ADJ_VECS = 2;                                // groups of 8 columns a thread
constexpr int ADJ_CHUNK = ADJ_THREADS * ADJ_VECS * 8;  // columns a block

// z / r as z * (1 / r): a rounding of 2^-24 more
__device__ __forceinline__ float adjusted(float x, uint32_t c, float r, float inv_r, float f, float p) {
  if (c) {
    const int made = c & 0x7FFF;
    x *= x > 0.f ? inv_r : r;
    if (made) x -= fmaf(f, (float)made, p);
  }
  return x;
}

// 4 bits -> 4 bytes of 0xFF or 0
__device__ __forceinline__ uint32_t spread4(uint32_t bits) {
  return ((bits & 0xFu) * 0x00204081u & 0x01010101u) * 0xFFu;
}

// grid (chunks of the vocabulary, rows).  Bound by HBM: 6 bytes and a bit read or
// written per bf16 logit, and 6 bytes a column leave no room for 40 instructions a
// column: the logits stay packed, and only pairs of columns with a count or a bias are
// taken apart (1 % of the columns are seen or biased in a request of some thousand
// tokens: 40 % of a warp's pairs).  256 rows of 128256 with 300 biases each and masks
// in %ADJ%.
// VEC: every row of every table starts on 16 bytes; a thread takes 8 neighbouring
// columns at a time.  Otherwise (an odd vocabulary without a padded pitch) its 8 lie a
// block's width apart, one access each.
template <typename T, bool VEC>
__global__ void __launch_bounds__(ADJ_THREADS) adjust_logits_kernel(LkAdjustLogitsDesc d) {
  constexpr bool F32 = sizeof(T) == 4;
  __shared__ float extra[ADJ_CHUNK];               // the row's biases in this chunk
  __shared__ uint32_t biased[ADJ_CHUNK / 32];      // which columns have one
  const int i = blockIdx.y, tid = threadIdx.x, v0 = blockIdx.x * ADJ_CHUNK, n = min(ADJ_CHUNK, d.vocab - v0);
  const T* in = (const T*)d.logits + (int64_t)i * d.ld + v0;
  T* out = (T*)d.out + (int64_t)i * d.ldo + v0;
  int row = d.counts ? (d.rows ? d.rows[i] : i) : -1;
  int mrow = d.mask ? (d.mask_rows ? d.mask_rows[i] : i) : -1;
  const int b0 = d.bias_offsets ? max(0, d.bias_offsets[i]) : 0, b1 = d.bias_offsets ? min(d.bias_count, d.bias_offsets[i + 1]) : 0;
  if (row >= d.count_rows || mrow >= d.mask_count) {
    if (tid == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    if (row >= d.count_rows) row = -1;
    if (mrow >= d.mask_count) mrow = -1;
  }
  const int16_t* counts = d.counts + (row >= 0 ? row * d.ldc + v0 : 0);
  const int* mask = d.mask + (mrow >= 0 ? mrow * d.ldm + v0 / 32 : 0);  // v0 is a multiple of 32
  // column k of this thread's group g
  auto col = [&](int g, int k) { return VEC ? (g * ADJ_THREADS + tid) * 8 + k : (g * 8 + k) * ADJ_THREADS + tid; };

  // everything is loaded first: x holds pairs of bf16 or single floats, c pairs of counts
  uint32_t x[ADJ_VECS][F32 ? 8 : 4], c[ADJ_VECS][4], allowed[ADJ_VECS];
#pragma unroll
  for (int g = 0; g < ADJ_VECS; ++g) {
    if (VEC && col(g, 0) + 8 <= n) {
#pragma unroll
      for (int q = 0; q < (F32 ? 2 : 1); ++q) {
        const uint4 a = reinterpret_cast<const uint4*>(in + col(g, 0))[q];
        x[g][4 * q] = a.x, x[g][4 * q + 1] = a.y, x[g][4 * q + 2] = a.z, x[g][4 * q + 3] = a.w;
      }
      uint4 a = make_uint4(0, 0, 0, 0);
      if (row >= 0) a = *reinterpret_cast<const uint4*>(counts + col(g, 0));
      c[g][0] = a.x, c[g][1] = a.y, c[g][2] = a.z, c[g][3] = a.w;
      allowed[g] = mrow >= 0 ? reinterpret_cast<const uint8_t*>(mask)[col(g, 0) / 8] : 0xFFu;
    } else {
      allowed[g] = 0;
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        uint32_t xw[2] = {0, 0}, cw[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int j = col(g, k + q);
          if (j < n) {
            if constexpr (F32) xw[q] = __float_as_uint(in[j]);
            else xw[q] = __bfloat16_as_ushort(in[j]);
            if (row >= 0) cw[q] = (uint16_t)counts[j];
            if (mrow < 0 || (mask[j / 32] >> (j & 31) & 1)) allowed[g] |= 1u << (k + q);
          }
        }
        if constexpr (F32) x[g][k] = xw[0], x[g][k + 1] = xw[1];
        else x[g][k / 2] = xw[0] | xw[1] << 16;
        c[g][k / 2] = cw[0] | cw[1] << 16;
      }
    }
  }
  const float r = row >= 0 ? d.penalties[3 * i] : 1.f, f = row >= 0 ? d.penalties[3 * i + 1] : 0.f,
              p = row >= 0 ? d.penalties[3 * i + 2] : 0.f;

  int any = 0;  // a bias falls into this chunk
  if (b0 < b1) {
    for (int j = tid; j < ADJ_CHUNK / 4; j += ADJ_THREADS) reinterpret_cast<float4*>(extra)[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (tid < ADJ_CHUNK / 32) biased[tid] = 0;
    __syncthreads();
    for (int j = b0 + tid; j < b1; j += ADJ_THREADS) {
      const int id = d.bias_ids[j], at = id - v0;
      if ((unsigned)id >= (unsigned)d.vocab) {
        if (blockIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
      } else if (at >= 0 && at < n) {
        atomicAdd(&extra[at], d.bias_values[j]);
        atomicOr(&biased[at / 32], 1u << (at & 31));
        any = 1;
      }
    }
    any = __syncthreads_or(any);
  }

  const float inv_r = 1.f / r;
#pragma unroll
  for (int g = 0; g < ADJ_VECS; ++g) {
    uint32_t bias_bits = 0;
    if (any) {
      if constexpr (VEC) {
        bias_bits = reinterpret_cast<const uint8_t*>(biased)[col(g, 0) / 8];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) bias_bits |= (biased[col(g, k) / 32] >> (col(g, k) & 31) & 1) << k;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      if (c[g][k / 2] | (bias_bits >> k & 3)) {
        float y[2];
        if constexpr (F32) y[0] = __uint_as_float(x[g][k]), y[1] = __uint_as_float(x[g][k + 1]);
        else y[0] = __uint_as_float(x[g][k / 2] << 16), y[1] = __uint_as_float(x[g][k / 2] & 0xFFFF0000u);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          y[q] = adjusted(y[q], c[g][k / 2] >> (16 * q) & 0xFFFFu, r, inv_r, f, p);
          if (bias_bits >> (k + q) & 1) y[q] += extra[col(g, k + q)];
        }
        if constexpr (F32) x[g][k] = __float_as_uint(y[0]), x[g][k + 1] = __float_as_uint(y[1]);
        else x[g][k / 2] = pack_bf16x2(y[0], y[1]);
      }
    }
    if (mrow >= 0) {
      if constexpr (F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (!(allowed[g] >> k & 1)) x[g][k] = 0xFF800000u;
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t keep = spread4(allowed[g] >> (4 * q));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t m = __byte_perm(keep, 0, k ? 0x3322 : 0x1100);
            x[g][2 * q + k] = (x[g][2 * q + k] & m) | (~m & 0xFF80FF80u);
          }
        }
      }
    }
    if (VEC && col(g, 0) + 8 <= n) {
#pragma unroll
      for (int q = 0; q < (F32 ? 2 : 1); ++q)
        reinterpret_cast<uint4*>(out + col(g, 0))[q] = make_uint4(x[g][4 * q], x[g][4 * q + 1], x[g][4 * q + 2], x[g][4 * q + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col(g, k) < n) {
          if constexpr (F32) out[col(g, k)] = __uint_as_float(x[g][k]);
          else out[col(g, k)] = __ushort_as_bfloat16((unsigned short)(x[g][k / 2] >> (16 * (k & 1))));
        }
    }
  }
}

constexpr int CNT_THREADS = 512;
constexpr int CNT_CHUNK = 8192;  // vocabulary columns per block (a 32 KB histogram)

// grid (chunks, sequences): histogram of a sequence's history over the block's
// vocabulary columns in shared memory, written over the row.  Every chunk reads the
// whole history (from L2 after the first); integer adds, so their order does not matter.
__global__ void __launch_bounds__(CNT_THREADS) set_token_counts_kernel(LkTokenCountsDesc d, bool vec) {
  __shared__ __align__(16) uint32_t hist[CNT_CHUNK];
  const int i = blockIdx.y, v0 = blockIdx.x * CNT_CHUNK, n = min(CNT_CHUNK, d.vocab - v0);
  const int row = d.rows ? d.rows[i] : i;
  if (row < 0 || row >= d.count_rows) {
    if (row >= d.count_rows && threadIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    return;
  }
  const int a = max(0, d.offsets[i]), b = min(d.num_tokens, d.offsets[i + 1]);
  const int64_t prompt = (int64_t)a + d.prompt_lens[i];
  for (int j = threadIdx.x; j < CNT_CHUNK / 4; j += CNT_THREADS) reinterpret_cast<uint4*>(hist)[j] = make_uint4(0, 0, 0, 0);
  __syncthreads();
#pragma unroll 4
  for (int k = a + threadIdx.x; k < b; k += CNT_THREADS) {
    const int64_t id = d.tokens[k];
    if (id < 0 || id >= d.vocab) {
      if (blockIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    } else if (id >= v0 && id < v0 + n) {
      if (k < prompt) atomicOr(&hist[id - v0], 0x80000000u);
      else atomicAdd(&hist[id - v0], 1u);
    }
  }
  __syncthreads();
  int16_t* out = d.counts + (int64_t)row * d.ldc + v0;
  auto packed = [&](int j) {
    const uint32_t c = hist[j];
    return min(c & 0x7FFFFFFFu, 32767u) | (c >> 31 << 15);
  };
  for (int j = threadIdx.x * 8; j < n; j += CNT_THREADS * 8) {
    if (vec && j + 8 <= n) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = packed(j + 2 * k) | packed(j + 2 * k + 1) << 16;
      *reinterpret_cast<uint4*>(out + j) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int k = j; k < min(j + 8, n); ++k) out[k] = (int16_t)packed(k);
    }
  }
}

// One thread per (row, token): the 16-bit count in its 32-bit word, saturating.
__global__ void add_token_counts_kernel(int16_t* counts, int64_t ldc, int count_rows, int vocab, const int* rows,
                                        const int64_t* tokens, int n, int* status) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const int row = rows ? rows[i] : i;
  if (row < 0) return;
  const int64_t id = tokens[i];
  if (row >= count_rows || id < 0 || id >= vocab) {
    if (status) atomicCAS(status, 0, LK_ERR_BAD_INDEX);
    return;
  }
  unsigned short* at = reinterpret_cast<unsigned short*>(counts + (int64_t)row * ldc + id);
  unsigned short seen = *at;
  while ((seen & 0x7FFF) != 0x7FFF) {
    const unsigned short was = atomicCAS(at, seen, (unsigned short)(seen + 1));
    if (was == seen) break;
    seen = was;
  }
}

// rows of `pitch` elements of `bytes` from p all start on 16 bytes
static bool rows_aligned(const void* p, int64_t pitch, int bytes, int rows) {
  return (uintptr_t)p % 16 == 0 && (rows <= 1 || pitch * bytes % 16 == 0);
}

}  // namespace lk

using namespace lk;

extern "C" int lk_adjust_logits(const LkAdjustLogitsDesc* d, cudaStream_t s) {
  if (d->n == 0 || d->vocab == 0) return 0;
  LK_REQUIRE(d->n <= 65535, "adjust_logits: at most 65535 rows");
  const dim3 grid(cdiv(d->vocab, ADJ_CHUNK), d->n);
  const int each = d->f32 ? 4 : 2;
  const bool vec = rows_aligned(d->logits, d->ld, each, d->n) && rows_aligned(d->out, d->ldo, each, d->n) &&
                   (!d->counts || rows_aligned(d->counts, d->ldc, 2, d->count_rows));
  if (d->f32)
    vec ? adjust_logits_kernel<float, true><<<grid, ADJ_THREADS, 0, s>>>(*d)
        : adjust_logits_kernel<float, false><<<grid, ADJ_THREADS, 0, s>>>(*d);
  else
    vec ? adjust_logits_kernel<__nv_bfloat16, true><<<grid, ADJ_THREADS, 0, s>>>(*d)
        : adjust_logits_kernel<__nv_bfloat16, false><<<grid, ADJ_THREADS, 0, s>>>(*d);
  return check_launch("adjust_logits");
}

extern "C" int lk_set_token_counts(const LkTokenCountsDesc* d, cudaStream_t s) {
  if (d->n == 0 || d->vocab == 0) return 0;
  LK_REQUIRE(d->n <= 65535, "set_token_counts: at most 65535 rows");
  set_token_counts_kernel<<<dim3(cdiv(d->vocab, CNT_CHUNK), d->n), CNT_THREADS, 0, s>>>(
      *d, rows_aligned(d->counts, d->ldc, 2, d->count_rows));
  return check_launch("set_token_counts");
}

extern "C" int lk_add_token_counts(int16_t* counts, int64_t ldc, int count_rows, int vocab, const int* rows,
                                   const int64_t* tokens, int n, int* status, cudaStream_t s) {
  if (n == 0) return 0;
  add_token_counts_kernel<<<cdiv(n, 128), 128, 0, s>>>(counts, ldc, count_rows, vocab, rows, tokens, n, status);
  return check_launch("add_token_counts");
}
