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

template <typename T>
__device__ __forceinline__ float logit_in(T x);
template <>
__device__ __forceinline__ float logit_in<float>(float x) { return x; }
template <>
__device__ __forceinline__ float logit_in<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T logit_out(float x);
template <>
__device__ __forceinline__ float logit_out<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 logit_out<__nv_bfloat16>(float x) { return __float2bfloat16(x); }

constexpr int ADJ_THREADS = 256;
constexpr int ADJ_CHUNK = 2048;  // vocabulary columns per block

// grid (chunks, rows)
template <typename T>
__global__ void __launch_bounds__(ADJ_THREADS) adjust_logits_kernel(LkAdjustLogitsDesc d) {
  __shared__ float z[ADJ_CHUNK];
  const int i = blockIdx.y, v0 = blockIdx.x * ADJ_CHUNK, n = min(ADJ_CHUNK, d.vocab - v0);
  const T* in = (const T*)d.logits + (int64_t)i * d.ld + v0;
  T* out = (T*)d.out + (int64_t)i * d.ldo + v0;
  int row = d.counts ? (d.rows ? d.rows[i] : i) : -1;
  if (row >= d.count_rows) {
    if (threadIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    row = -1;
  }
  const float r = row >= 0 ? d.penalties[3 * i] : 1.f, f = row >= 0 ? d.penalties[3 * i + 1] : 0.f,
              p = row >= 0 ? d.penalties[3 * i + 2] : 0.f;
  for (int j = threadIdx.x; j < n; j += ADJ_THREADS) {
    float x = logit_in<T>(in[j]);
    const int c = row >= 0 ? (int)(uint16_t)d.counts[(int64_t)row * d.ldc + v0 + j] : 0;
    if (c) {
      const int made = c & 0x7FFF;
      x = x > 0.f ? x / r : x * r;
      if (made) x = x - f * made - p;
    }
    z[j] = x;
  }
  __syncthreads();
  if (d.bias_offsets) {
    const int a = max(0, d.bias_offsets[i]), b = min(d.bias_count, d.bias_offsets[i + 1]);
    for (int k = a + threadIdx.x; k < b; k += ADJ_THREADS) {
      const int id = d.bias_ids[k];
      if (id < 0 || id >= d.vocab) {
        if (blockIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
      } else if (id >= v0 && id < v0 + n) {
        atomicAdd(&z[id - v0], d.bias_values[k]);
      }
    }
    __syncthreads();
  }
  int mrow = d.mask ? (d.mask_rows ? d.mask_rows[i] : i) : -1;
  if (mrow >= d.mask_count) {
    if (threadIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    mrow = -1;
  }
  const int* mask = d.mask + (int64_t)max(mrow, 0) * d.ldm;
  for (int j = threadIdx.x; j < n; j += ADJ_THREADS) {
    const bool allowed = mrow < 0 || ((mask[(v0 + j) >> 5] >> ((v0 + j) & 31)) & 1);
    out[j] = logit_out<T>(allowed ? z[j] : -INFINITY);
  }
}

constexpr int CNT_CHUNK = 8192;  // vocabulary columns per block (a 32 KB histogram)

// grid (chunks, sequences): histogram of a sequence's history over the block's
// vocabulary columns in shared memory, written over the row.
__global__ void __launch_bounds__(256) set_token_counts_kernel(LkTokenCountsDesc d) {
  __shared__ uint32_t hist[CNT_CHUNK];
  const int i = blockIdx.y, v0 = blockIdx.x * CNT_CHUNK, n = min(CNT_CHUNK, d.vocab - v0);
  const int row = d.rows ? d.rows[i] : i;
  if (row < 0 || row >= d.count_rows) {
    if (row >= d.count_rows && threadIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    return;
  }
  for (int j = threadIdx.x; j < n; j += 256) hist[j] = 0;
  __syncthreads();
  const int a = max(0, d.offsets[i]), b = min(d.num_tokens, d.offsets[i + 1]);
  const int prompt = a + d.prompt_lens[i];
  for (int k = a + threadIdx.x; k < b; k += 256) {
    const int64_t id = d.tokens[k];
    if (id < 0 || id >= d.vocab) {
      if (blockIdx.x == 0 && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
    } else if (id >= v0 && id < v0 + n) {
      if (k < prompt) atomicOr(&hist[id - v0], 0x80000000u);
      else atomicAdd(&hist[id - v0], 1u);
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += 256) {
    const uint32_t c = hist[j];
    d.counts[(int64_t)row * d.ldc + v0 + j] = (int16_t)(min(c & 0x7FFFFFFFu, 32767u) | (c >> 31 << 15));
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

}  // namespace lk

using namespace lk;

extern "C" int lk_adjust_logits(const LkAdjustLogitsDesc* d, cudaStream_t s) {
  if (d->n == 0 || d->vocab == 0) return 0;
  LK_REQUIRE(d->n <= 65535, "adjust_logits: at most 65535 rows");
  const dim3 grid(cdiv(d->vocab, ADJ_CHUNK), d->n);
  d->f32 ? adjust_logits_kernel<float><<<grid, ADJ_THREADS, 0, s>>>(*d)
         : adjust_logits_kernel<__nv_bfloat16><<<grid, ADJ_THREADS, 0, s>>>(*d);
  return check_launch("adjust_logits");
}

extern "C" int lk_set_token_counts(const LkTokenCountsDesc* d, cudaStream_t s) {
  if (d->n == 0 || d->vocab == 0) return 0;
  LK_REQUIRE(d->n <= 65535, "set_token_counts: at most 65535 rows");
  set_token_counts_kernel<<<dim3(cdiv(d->vocab, CNT_CHUNK), d->n), 256, 0, s>>>(*d);
  return check_launch("set_token_counts");
}

extern "C" int lk_add_token_counts(int16_t* counts, int64_t ldc, int count_rows, int vocab, const int* rows,
                                   const int64_t* tokens, int n, int* status, cudaStream_t s) {
  if (n == 0) return 0;
  add_token_counts_kernel<<<cdiv(n, 128), 128, 0, s>>>(counts, ldc, count_rows, vocab, rows, tokens, n, status);
  return check_launch("add_token_counts");
}
