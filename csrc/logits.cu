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
constexpr int ADJ_STEP = ADJ_THREADS * 8;  // columns a block takes with one group of 8 a thread
constexpr int ADJ_GROUPS = 2;              // groups a thread takes where there are many rows

// z / r as z * (1 / r): a rounding of 2^-24 more.  Without branches; a token not seen
// (c = 0) keeps its bits (x * 1 - 0).
__device__ __forceinline__ float adjusted(float x, uint32_t c, float r, float inv_r, float f, float p) {
  const uint32_t made = c & 0x7FFFu;
  const float scale = c ? (x > 0.f ? inv_r : r) : 1.f;
  return fmaf(x, scale, made ? -fmaf(f, (float)made, p) : -0.f);
}

// 4 bits -> 4 bytes of 0xFF or 0
__device__ __forceinline__ uint32_t spread4(uint32_t bits) {
  return ((bits & 0xFu) * 0x00204081u & 0x01010101u) * 0xFFu;
}

// 8 columns of a row as loaded: pairs of bf16 or single floats, pairs of counts, mask bits
template <bool F32>
struct AdjGroup {
  uint32_t x[F32 ? 8 : 4], c[4], allowed;
};

// grid (spans of the vocabulary, rows); a thread's G groups of 8 columns are all loaded
// before anything else, which is what keeps enough bytes on their way.  Bound by HBM: 6 bytes and
// a bit read or written per bf16 logit, which leaves no room for 40 instructions a
// column: the logits stay packed, and only pairs of columns with a count or a bias are
// taken apart (1 % of the columns are seen or biased in a request of some thousand
// tokens: 40 % of a warp's pairs).  256 rows of 128256 with 300 biases each and masks
// in 38.9 us, 35 without biases (torch.add of the logits and the counts: 31); 1 or 4 groups,
// 5 blocks an SM and blocks of 512 are 2-15 us slower.
// VEC: every row of every table starts on 16 bytes; a thread takes 8 neighbouring
// columns at a time.  Otherwise (an odd vocabulary without a padded pitch) its 8 lie a
// block's width apart, one access each: 128 rows of 128251 in 44 us, of 128256 in 20.
template <typename T, bool VEC, int G>
__global__ void __launch_bounds__(ADJ_THREADS, G == 1 || (VEC && sizeof(T) == 2) ? 6 : 3) adjust_logits_kernel(LkAdjustLogitsDesc d) {
  constexpr bool F32 = sizeof(T) == 4;
  extern __shared__ __align__(16) float extra[];  // the row's biases in this span, then a bit per column that has one
  uint32_t* biased = reinterpret_cast<uint32_t*>(extra + G * ADJ_STEP);
  const int i = blockIdx.y, tid = threadIdx.x, v0 = blockIdx.x * G * ADJ_STEP, n = min(G * ADJ_STEP, d.vocab - v0);
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
  // column k of this thread in the group that begins at column s
  auto col = [&](int s, int k) { return s + (VEC ? tid * 8 + k : k * ADJ_THREADS + tid); };
  auto load = [&](int s) {
    AdjGroup<F32> g;
    if (VEC && col(s, 0) + 8 <= n) {
#pragma unroll
      for (int q = 0; q < (F32 ? 2 : 1); ++q) {
        const uint4 a = reinterpret_cast<const uint4*>(in + col(s, 0))[q];
        g.x[4 * q] = a.x, g.x[4 * q + 1] = a.y, g.x[4 * q + 2] = a.z, g.x[4 * q + 3] = a.w;
      }
      uint4 a = make_uint4(0, 0, 0, 0);
      if (row >= 0) a = *reinterpret_cast<const uint4*>(counts + col(s, 0));
      g.c[0] = a.x, g.c[1] = a.y, g.c[2] = a.z, g.c[3] = a.w;
      g.allowed = mrow >= 0 ? reinterpret_cast<const uint8_t*>(mask)[col(s, 0) / 8] : 0xFFu;
    } else if (VEC) {  // the end of a row
      g.allowed = 0;
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        uint32_t xw[2] = {0, 0}, cw[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int j = col(s, k + q);
          if (j < n) {
            if constexpr (F32) xw[q] = __float_as_uint(in[j]);
            else xw[q] = __bfloat16_as_ushort(in[j]);
            if (row >= 0) cw[q] = (uint16_t)counts[j];
            if (mrow < 0 || (mask[j / 32] >> (j & 31) & 1)) g.allowed |= 1u << (k + q);
          }
        }
        if constexpr (F32) g.x[k] = xw[0], g.x[k + 1] = xw[1];
        else g.x[k / 2] = xw[0] | xw[1] << 16;
        g.c[k / 2] = cw[0] | cw[1] << 16;
      }
    } else {
      // columns past the end ask for the last one again: no branch between the loads
      uint32_t x[8], c[8], w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = min(col(s, k), n - 1);
        if constexpr (F32) x[k] = __float_as_uint(in[j]);
        else x[k] = __bfloat16_as_ushort(in[j]);
        c[k] = row >= 0 ? (uint16_t)counts[j] : 0;
        w[k] = mrow >= 0 ? (uint32_t)mask[j / 32] : ~0u;
      }
      g.allowed = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        g.allowed |= (w[k] >> (col(s, k) & 31) & 1) << k;
        if (k & 1) g.c[k / 2] = c[k - 1] | c[k] << 16;
        if constexpr (F32) g.x[k] = x[k];
        else if (k & 1) g.x[k / 2] = x[k - 1] | x[k] << 16;
      }
    }
    return g;
  };
  AdjGroup<F32> groups[G];
#pragma unroll
  for (int s = 0; s < G; ++s) groups[s] = load(s * ADJ_STEP);
  const float r = row >= 0 ? d.penalties[3 * i] : 1.f, f = row >= 0 ? d.penalties[3 * i + 1] : 0.f,
              p = row >= 0 ? d.penalties[3 * i + 2] : 0.f;

  int any = 0;  // a bias falls into this span
  __shared__ int again;  // two biases fall onto one column
  if (b0 < b1) {
    // ids and values of a thread's first two biases are asked for together and at once:
    // the block lives as long as its longest chain of loads
    constexpr int FIRST = 2;
    int id[FIRST];
    float value[FIRST];
#pragma unroll
    for (int k = 0; k < FIRST; ++k) {
      const int j = b0 + tid + k * ADJ_THREADS;
      id[k] = j < b1 ? d.bias_ids[j] : v0;
      value[k] = j < b1 ? d.bias_values[j] : 0.f;
    }
    constexpr int words = G * (ADJ_STEP + ADJ_STEP / 32) / 4;
    for (int j = tid; j < words; j += ADJ_THREADS) reinterpret_cast<float4*>(extra)[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (tid == 0) again = 0;
    __syncthreads();
    auto add = [&](int token, float x) {
      const int at = token - v0;
      if ((unsigned)at < (unsigned)n) {
        const uint32_t bit = 1u << (at & 31);
        if (atomicOr(&biased[at / 32], bit) & bit) again = 1;
        else extra[at] = x;
        any = 1;
      } else if (blockIdx.x == 0 && (unsigned)token >= (unsigned)d.vocab && d.status) {
        atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
      }
    };
#pragma unroll
    for (int k = 0; k < FIRST; ++k)
      if (b0 + tid + k * ADJ_THREADS < b1) add(id[k], value[k]);
    for (int j = b0 + tid + FIRST * ADJ_THREADS; j < b1; j += ADJ_THREADS) add(d.bias_ids[j], d.bias_values[j]);
    any = __syncthreads_or(any);
    if (again) {  // an id is named more than once: each thread adds up its own columns in the list's order
#pragma unroll 1
      for (int j = tid; j < G * ADJ_STEP; j += ADJ_THREADS) extra[j] = 0.f;
#pragma unroll 1
      for (int j = b0; j < b1; ++j) {
        const int at = d.bias_ids[j] - v0;
        if ((unsigned)at < (unsigned)n && at % ADJ_THREADS == tid) extra[at] += d.bias_values[j];
      }
      __syncthreads();
    }
  }

  const float inv_r = 1.f / r;
#pragma unroll
  for (int e = 0; e < G; ++e) {
    const int s = e * ADJ_STEP;
    AdjGroup<F32>& g = groups[e];
    uint32_t bias_bits = 0;
    if (any) {
      if constexpr (VEC) {
        bias_bits = reinterpret_cast<const uint8_t*>(biased)[col(s, 0) / 8];
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) bias_bits |= (biased[col(s, k) / 32] >> (col(s, k) & 31) & 1) << k;
      }
    }
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      if (g.c[k / 2] | (bias_bits >> k & 3)) {
        float y[2];
        if constexpr (F32) y[0] = __uint_as_float(g.x[k]), y[1] = __uint_as_float(g.x[k + 1]);
        else y[0] = __uint_as_float(g.x[k / 2] << 16), y[1] = __uint_as_float(g.x[k / 2] & 0xFFFF0000u);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          y[q] = adjusted(y[q], g.c[k / 2] >> (16 * q) & 0xFFFFu, r, inv_r, f, p);
          if (bias_bits >> (k + q) & 1) y[q] += extra[col(s, k + q)];
        }
        if constexpr (F32) g.x[k] = __float_as_uint(y[0]), g.x[k + 1] = __float_as_uint(y[1]);
        else g.x[k / 2] = pack_bf16x2(y[0], y[1]);
      }
    }
    if (mrow >= 0) {
      if constexpr (F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (!(g.allowed >> k & 1)) g.x[k] = 0xFF800000u;
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t keep = spread4(g.allowed >> (4 * q));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t m = __byte_perm(keep, 0, k ? 0x3322 : 0x1100);
            g.x[2 * q + k] = (g.x[2 * q + k] & m) | (~m & 0xFF80FF80u);
          }
        }
      }
    }
    if (VEC && col(s, 0) + 8 <= n) {
#pragma unroll
      for (int q = 0; q < (F32 ? 2 : 1); ++q)
        reinterpret_cast<uint4*>(out + col(s, 0))[q] = make_uint4(g.x[4 * q], g.x[4 * q + 1], g.x[4 * q + 2], g.x[4 * q + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col(s, k) < n) {
          if constexpr (F32) out[col(s, k)] = __uint_as_float(g.x[k]);
          else out[col(s, k)] = __ushort_as_bfloat16((unsigned short)(g.x[k / 2] >> (16 * (k & 1))));
        }
    }
  }
}

constexpr int CNT_THREADS = 512;
constexpr int CNT_CHUNK = 4096;  // vocabulary columns per block (a 16 KB histogram)

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
  if (vec) {
    for (int j = threadIdx.x * 8; j < n; j += CNT_THREADS * 8) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = packed(j + 2 * k) | packed(j + 2 * k + 1) << 16;
      if (j + 8 <= n) *reinterpret_cast<uint4*>(out + j) = make_uint4(w[0], w[1], w[2], w[3]);
      else for (int k = j; k < n; ++k) out[k] = (int16_t)packed(k);
    }
  } else {
    for (int j = threadIdx.x; j < n; j += CNT_THREADS) out[j] = (int16_t)packed(j);
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
  const int each = d->f32 ? 4 : 2;
  const bool vec = rows_aligned(d->logits, d->ld, each, d->n) && rows_aligned(d->out, d->ldo, each, d->n) &&
                   (!d->counts || rows_aligned(d->counts, d->ldc, 2, d->count_rows));
  // two groups a thread share the search for a row's biases and have more loads on their way,
  // one fills the GPU sooner (us with 1 / 2 groups, 300 biases a row, 128256 columns: 1 row 2.8 /
  // 2.9, 16 rows 4.9 / 4.3, 48 rows 9.8 / 8.0; 128251 columns: 3.1 / 4.1, 7.7 / 7.7, 18.2 / 17.0)
  const int groups = (int64_t)d->n * cdiv(d->vocab, ADJ_GROUPS * ADJ_STEP) >= 2 * num_sms() ? ADJ_GROUPS : 1;
  const dim3 grid(cdiv(d->vocab, groups * ADJ_STEP), d->n);
  const int smem = d->bias_offsets ? groups * (ADJ_STEP + ADJ_STEP / 32) * 4 : 0;
#define LK_ADJ(T, VEC)                                                                           \
  (groups == 1 ? adjust_logits_kernel<T, VEC, 1><<<grid, ADJ_THREADS, smem, s>>>(*d)             \
               : adjust_logits_kernel<T, VEC, ADJ_GROUPS><<<grid, ADJ_THREADS, smem, s>>>(*d))
  if (d->f32) vec ? LK_ADJ(float, true) : LK_ADJ(float, false);
  else vec ? LK_ADJ(__nv_bfloat16, true) : LK_ADJ(__nv_bfloat16, false);
#undef LK_ADJ
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
