// Attention of the newest q_len tokens of each sequence over the page-scaled
// 8-bit KV cache (csrc/kv_page.cu describes the cache).
//
//   s[t] = (q . k[t]) * scale * kscale[page(t)],  t <= position of the query
//   out  = sum_t softmax(s)[t] * v[t] * vscale[page(t)]
//
// Query j of a sequence of ctx tokens sits at position ctx - q_len + j.  A query
// without a token before it (an unused batch row of ctx 0) gives zeros.
//
// The cache is read once per tile of 8 or 16 query rows: 2 * Hkv * Dh bytes a token, against
// 4 * Hq * Dh flops per query token, so HBM bounds it as long as the work per byte stays small.
// On CUDA cores it does not (conversions, products and the reductions of the
// scores cost more issue slots than the bytes bring), hence tensor cores, with
// the tokens as the M dimension of both products so that the few query rows
// (GQA group * q_len, columns of 8) waste nothing:
//
//   S^T [tokens x queries] = K Q^T      O^T [dims x queries] += V^T P^T
//
// mma.sync m16n8k16 in f16 with fp32 sums: a code is exact in f16 (e4m3 by one
// conversion per two codes), and the fragments of K and of V^T are exactly what
// 16-byte loads of the cached rows bring to each lane, the order of the
// summed index being free (dims for K; a lane's dims are 16 neighbours of one
// row).  tcgen05 would want both operands in 8 bits (the query rounded to them)
// or the codes converted into shared memory first.  Each warp fills a ring of its
// own with cp.async: no barrier between warps, and addresses are free, so any page
// size works and a page may end inside a tile.
//
// Softmax per warp, one pass.  Weights are f16, so they are taken relative to
// a running reference m with 2^7 at the largest one so far and moved only when
// a score passes 2^14 (f16 ends at 2^16): weights down to 2^-31 of the largest
// count.  A page's value scale 2^e enters as e added to the score, with a
// reference of its own: a page of small values is then as exact as one of large
// ones whichever the query looks at.  The softmax sum is kept in fp32 apart.
//
// Measured: 256 sequences of up to 4096 tokens (32 / 8 heads of 128, e4m3, 1084 MB)
// 184-195 us, 85-90 % of the HBM copy rate; two of 100003 tokens 63-66 us (77-80 %); int8 codes
// take two instructions more a pair: 197 us.  A block costs 3.5 us beside its tokens
// (launch, length and pages, first data, merge), which is what the full batch lacks, and
// at head_dim 64 more (4 KV heads: 64 us for a floor of 42).  Where rows are few, a warp's 480
// instructions per 32 tokens and their dependences bound it: 24 sequences of up to 2047
// tokens with five queries each (40 rows, 8 / 1 heads of 64, int8) 22.5 us.
#include <algorithm>
#include <mutex>
#include <utility>

#include "common.cuh"
#include "host_util.h"
#include "kv_page.cuh"
#include "lk_api.h"

namespace lk {

constexpr int PA_WARPS = 4;
constexpr int PA_STAGES = 2;  // units on their way per warp (1 with 4 blocks an SM, 3 with 2: 7 to 15 % slower)
constexpr int PA_CLUSTER = 16;     // parts that one cluster of blocks joins
constexpr int PA_UNIT = 32;        // tokens a warp takes at a time (two M = 16 tiles)
constexpr float PA_LOW = -3.0e38f;  // reference before the first token
constexpr float PA_TOP = 14.f, PA_AIM = 7.f;

// A stage of a warp's ring: a unit's keys, values, scales and valid tokens.  Rows lie in
// 128-byte lines (a line holds two tokens where DH = 64) whose 16-byte chunks are
// exchanged by an XOR, so that the copies write whole lines and the fragment reads
// touch every bank once: keys, 8 lanes read chunks 0-3 (or 4-7) of tokens 2a and
// 2a + 1; values, 8 lanes read chunks 2b and 2b + 1 of tokens 0, 2, 4, 6 (or 1, 3, 5, 7)
// of a group of 8, 16 lanes 32 bytes of each where DH = 64.
template <int DH>
struct PaRing {
  static constexpr int KV_BYTES = PA_UNIT * DH;      // keys (or values) of a unit
  static constexpr int SCALES = 2 * KV_BYTES;        // float2 (key, value scale) per token
  static constexpr int MASK = SCALES + PA_UNIT * 8;  // bit per token: its page id is valid
  static constexpr int STAGE = (MASK + 4 + 127) / 128 * 128;
  static constexpr int STAGES = PA_STAGES;
  static constexpr int WARP = STAGE * STAGES;
  // byte position of chunk k of token t
  static __device__ __forceinline__ uint32_t at(int t, int k) {
    if constexpr (DH == 128) return t * 128 + ((k ^ (t & 6) ^ ((t & 1) << 2)) << 4);
    else return (t >> 1) * 128 + ((((t & 1) << 2 | k) ^ (t & 6)) << 4);
  }
  // the token of the unit that a lane copies a chunk of with its copy i, and where to: i * 512
  // and what the lane and the parity of i say (at head_dim 64 the lane alone)
  static constexpr int LANES = DH / 16;  // lanes per row
  static __device__ __forceinline__ int token(int i, int lane) { return i * (32 / LANES) + lane / LANES; }
  static __device__ __forceinline__ uint32_t place(int odd, int lane) { return at(token(odd, lane), lane % LANES) - odd * 512; }
};

// 16 bytes to shared address dst + OFF (a constant that stays in the instruction);
// or zeros, with nothing read.
template <int OFF>
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
}
template <int OFF>
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1], 16, %3;" ::"r"(dst), "l"(src), "n"(OFF), "r"(on ? 16 : 0) : "memory");
}
template <typename F, int... I>
__device__ __forceinline__ void static_for_each(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>  // f(0), ..., f(N - 1), each argument a constant
__device__ __forceinline__ void static_for(F f) {
  static_for_each(f, std::make_integer_sequence<int, N>{});
}
// p + n * stride bytes in one multiply-add
template <typename T>
__device__ __forceinline__ const T* advance(const T* p, uint32_t n, uint32_t stride) {
  const T* q;
  asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(q) : "r"(n), "r"(stride), "l"(p));
  return q;
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(addr));
  return x;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr));
  return x;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Codes of the low (HI = 0) or high two bytes of w as f16x2.  int8: byte ^ 0x80
// under the exponent of 1024 is 1152 + code.
template <int KV, int HI>
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t w) {
  if constexpr (KV == 1) {
    uint32_t h;
    if constexpr (HI) asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}\n" : "=r"(h) : "r"(w));
    else asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(h) : "r"(w));
    return h;
  } else {
    const uint32_t u = __byte_perm(w ^ 0x80808080u, 0x64646464u, HI ? 0x4342 : 0x4140);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// What the blocks of a sequence's row tile share: the tokens [0, end) that any of
// its queries sees, cut into at most nsplit parts of `per` units.
struct PaSpan {
  int ctx, end, units, per;
};

__device__ __forceinline__ PaSpan page_attn_span(const LkPageAttnDesc& d, int ctx, int last_token) {
  PaSpan s;
  s.ctx = (int)min((int64_t)max(ctx, 0), (int64_t)d.max_pages * d.page);
  s.end = max(0, s.ctx - d.q_len + last_token + 1);
  s.units = (s.end + PA_UNIT - 1) / PA_UNIT;
  s.per = max((s.units + d.nsplit - 1) / d.nsplit, PA_WARPS);  // a unit for each warp at least
  return s;
}

struct PaDivs {
  FastDiv nsplit, heads, tiles, group, page;
};

// Grid: split fastest, then KV head, row tile (8 * NT query rows), sequence.
template <int KV, int DH, int NT>
__global__ void __launch_bounds__(32 * PA_WARPS, NT == 1 ? (DH == 64 ? 4 : 3) : (DH == 64 ? 3 : 2)) page_attn_kernel(LkPageAttnDesc d, PaDivs by) {
  const int nsplit = d.nsplit, tiles = by.tiles.d;
  using R = PaRing<DH>;
  constexpr int ROWS = 8 * NT, CH = DH / 64, MT = DH / 16;
  extern __shared__ __align__(16) uint8_t sm[];
  // divisions by multiplication: a dozen of them are a good part of a short block's time
  int b = by.nsplit.div(blockIdx.x);
  const int split = blockIdx.x - b * nsplit;
  int h = b;
  b = by.heads.div(b);
  h -= b * d.Hkv;
  const int seq = by.tiles.div(b), tile = b - seq * tiles;
  const int group = by.group.d, rows = group * d.q_len;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int ctx = d.ctx_lens[seq];
  const int* table = d.tables + (int64_t)seq * d.max_pages;
  struct Place {
    int page, row;  // page id and row in the page
  };
  auto page_of = [&](int u) {  // of this lane's token of unit u; anything beyond the context is not used
    const int t = u * PA_UNIT + lane, i = by.page.div(t);
    return Place{i < d.max_pages ? table[i] : 0, t - i * d.page};
  };
  // an uncut context begins at unit `warp` whatever its length: its pages are looked up
  // while the length is on its way
  Place pg[PA_STAGES + 1];
  if (nsplit == 1) {
#pragma unroll
    for (int s = 0; s <= PA_STAGES; ++s) pg[s] = page_of(warp + s * PA_WARPS);
  }
  // query fragments: column r of each tile, the dims of this lane's key bytes, times
  // a power of two of its own that brings the row's largest value to [2^14, 2^15): f16 then
  // holds a bf16 value exactly down to 2^-31 of it, and 2^-39 of it is the rounding
  uint32_t qf[NT][4 * CH][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int row = tile * ROWS + n * 8 + r;
    uint32_t (&w)[4 * CH][2] = qf[n];  // bf16 pairs first
#pragma unroll
    for (int i = 0; i < 8 * CH; ++i) w[i / 2][i % 2] = 0;
    if (row < rows) {
      const int token = by.group.div(row);
      const uint4* p = reinterpret_cast<const uint4*>((const __nv_bfloat16*)d.q + ((int64_t)seq * d.q_len + token) * d.ldq +
                                                      (h * group + row - token * group) * DH);
#pragma unroll
      for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint4 v = p[k * 8 + c * 2 + i];
          w[k * 4 + i * 2][0] = v.x, w[k * 4 + i * 2][1] = v.y, w[k * 4 + i * 2 + 1][0] = v.z, w[k * 4 + i * 2 + 1][1] = v.w;
        }
    }
  }

  const PaSpan sp = page_attn_span(d, ctx, by.group.div(min(rows, (tile + 1) * ROWS) - 1));
  if (threadIdx.x == 0 && ctx > (int64_t)d.max_pages * d.page && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
  const int u_end = min(sp.units, (split + 1) * sp.per);
  cudaTriggerProgrammaticLaunchCompletion();  // the join may be brought up; it waits for all of this grid
  const bool cluster = nsplit > 1 && nsplit <= PA_CLUSTER;  // the parts' blocks are a cluster and join by themselves
  if (!cluster && split > 0 && split * sp.per >= sp.units) return;
  int u = split * sp.per + warp;
  if (nsplit > 1) {
#pragma unroll
    for (int s = 0; s <= PA_STAGES; ++s) pg[s] = page_of(u + s * PA_WARPS);
  }

  // where this lane copies from, and this warp's ring
  const uint32_t tok_stride = (uint32_t)d.Hkv * DH;
  const uint8_t* kbase = (const uint8_t*)d.k_cache + h * DH + lane % R::LANES * 16;
  const uint8_t* vbase = (const uint8_t*)d.v_cache + h * DH + lane % R::LANES * 16;
  uint8_t* ring = sm + warp * R::WARP;
  const uint32_t ring_u = smem_u32(ring);

  // the unit's copies: this lane looks up token `lane`, then copies 16 bytes of its share
  // of the rows (8 lanes a 128-byte line, so that a request is a whole line); its token's
  // scales go to registers and into the stage when the unit's turn comes
  const float* ks = d.k_scale + h;
  const float* vs = d.v_scale + h;
  const uint32_t to[2] = {ring_u + R::place(0, lane), ring_u + R::place(1, lane)};
  auto issue = [&](int u, int stage, Place at, float2& scales) {
    if (u < u_end) {
      const bool there = u * PA_UNIT + lane < sp.end, ok = there && (unsigned)at.page < (unsigned)d.num_pages;
      const unsigned valid = __ballot_sync(0xffffffffu, ok);
      const uint32_t page = ok ? at.page : 0, slot = ok ? page * d.page + at.row : 0, st = stage * R::STAGE;
      scales = make_float2(*advance(ks, page, d.Hkv * 4), *advance(vs, page, d.Hkv * 4));
      if (lane == 0) asm volatile("st.shared.u32 [%0+%1], %2;" ::"r"(ring_u + st), "n"(R::MASK), "r"(valid) : "memory");
      if (valid == 0xffffffffu) {
        static_for<DH / 16>([&](auto i) {
          const uint32_t s = __shfl_sync(0xffffffffu, slot, R::token(i, lane));
          cp_async16<i * 512>(to[i & 1] + st, advance(kbase, s, tok_stride));
          cp_async16<i * 512 + R::KV_BYTES>(to[i & 1] + st, advance(vbase, s, tok_stride));
        });
      } else {  // the end of the context, or a bad page id: nothing is read there, zeros take its place
        if (there && !ok && d.status) atomicCAS(d.status, 0, LK_ERR_BAD_INDEX);
        static_for<DH / 16>([&](auto i) {
          const uint32_t s = __shfl_sync(0xffffffffu, slot, R::token(i, lane));
          const bool on = (valid >> R::token(i, lane)) & 1;
          cp_async16_or_zero<i * 512>(to[i & 1] + st, advance(kbase, s, tok_stride), on);
          cp_async16_or_zero<i * 512 + R::KV_BYTES>(to[i & 1] + st, advance(vbase, s, tok_stride), on);
        });
      }
    }
    cp_commit();
  };

  float2 scales[R::STAGES];  // of the units in flight, the next one first
#pragma unroll
  for (int s = 0; s < R::STAGES; ++s) issue(u + s * PA_WARPS, s, pg[s], scales[s]);
  Place pg_next = pg[R::STAGES];

  int lim[NT][2];
  float qfac[NT][2];  // of this lane's score columns 2c and 2c + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float amax = 0.f;  // of row r of the tile, whose dims its four lanes hold
#pragma unroll
    for (int i = 0; i < 8 * CH; ++i) {
      const float2 f = unpack_bf16x2(qf[n][i / 2][i % 2]);
      if (fabsf(f.x) <= 3.4028234e38f) amax = fmaxf(amax, fabsf(f.x));
      if (fabsf(f.y) <= 3.4028234e38f) amax = fmaxf(amax, fabsf(f.y));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = max((int)(__float_as_uint(amax) >> 23) - 127 - 14, -112);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    const float up = __uint_as_float((uint32_t)(127 + e) << 23) * (d.scale * 1.4426950408889634f);
#pragma unroll
    for (int q = 0; q < 2; ++q) qfac[n][q] = __shfl_sync(0xffffffffu, up, (2 * c + q) * 4);
#pragma unroll
    for (int k = 0; k < 4 * CH; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 f = unpack_bf16x2(qf[n][k][i]);
        const __half2 hv = __floats2half2_rn(f.x * down, f.y * down);
        qf[n][k][i] = *reinterpret_cast<const uint32_t*>(&hv);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = tile * ROWS + n * 8 + 2 * c + i;
      lim[n][i] = col < rows ? sp.ctx - d.q_len + by.group.div(col) + 1 : sp.end;
    }
  }
  const int open = sp.ctx - d.q_len + by.group.div(tile * ROWS) + 1;  // tokens that every query of the tile sees

  float acc[NT][MT][4], ms[NT][2], mw[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][j][i] = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) ms[n][i] = mw[n][i] = PA_LOW, l[n][i] = 0.f;
  }

  int stage = 0;
  for (; u < u_end; u += PA_WARPS) {
    uint8_t* st = ring + stage * R::STAGE;
    *reinterpret_cast<float2*>(st + R::SCALES + lane * 8) = scales[0];
    cp_wait<R::STAGES - 1>();
    __syncwarp();
    // scores of both 16-token tiles
    float s[2][NT][4];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[g][n][i] = 0.f;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const uint4 lo = *reinterpret_cast<const uint4*>(st + R::at(16 * g + r, 4 * k + c));
        const uint4 hi = *reinterpret_cast<const uint4*>(st + R::at(16 * g + r + 8, 4 * k + c));
        const uint32_t xs[4] = {lo.x, lo.y, lo.z, lo.w}, ys[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = codes_f16x2<KV, 0>(xs[i]), a1 = codes_f16x2<KV, 0>(ys[i]);
          const uint32_t a2 = codes_f16x2<KV, 1>(xs[i]), a3 = codes_f16x2<KV, 1>(ys[i]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(s[g][n], a0, a1, a2, a3, qf[n][4 * k + i][0], qf[n][4 * k + i][1]);
        }
      }
    }
    // scale, mask; the score plus the value scale's exponent is the weight's exponent
    float x[2][NT][4];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 sc = *reinterpret_cast<const float2*>(st + R::SCALES + (16 * g + 8 * i + r) * 8);
        const float lv = __log2f(sc.y);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            s[g][n][2 * i + q] *= sc.x * qfac[n][q];
            x[g][n][2 * i + q] = s[g][n][2 * i + q] + lv;
          }
      }
    const unsigned valid = *reinterpret_cast<const unsigned*>(st + R::MASK);
    if (valid != 0xffffffffu || (u + 1) * PA_UNIT > open) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int tl = 16 * g + 8 * i + r;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (u * PA_UNIT + tl >= lim[n][q] || !((valid >> tl) & 1)) s[g][n][2 * i + q] = x[g][n][2 * i + q] = -INFINITY;
        }
    }
    float sa[NT][2], xa[NT][2];
    bool move = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        sa[n][q] = fmaxf(fmaxf(s[0][n][q], s[0][n][2 + q]), fmaxf(s[1][n][q], s[1][n][2 + q]));
        xa[n][q] = fmaxf(fmaxf(x[0][n][q], x[0][n][2 + q]), fmaxf(x[1][n][q], x[1][n][2 + q]));
        move |= sa[n][q] > ms[n][q] + PA_TOP || xa[n][q] > mw[n][q] + PA_TOP;
      }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float a = sa[n][q], w = xa[n][q];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, o));
          }
          // a column moves by its own scores alone: its bits do not depend on its neighbours
          if (a > ms[n][q] + PA_TOP) {
            l[n][q] *= fast_exp2(ms[n][q] - (a - PA_AIM));
            ms[n][q] = a - PA_AIM;
          }
          if (w > mw[n][q] + PA_TOP) {
            const float f = fast_exp2(mw[n][q] - (w - PA_AIM));
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[n][j][q] *= f, acc[n][j][2 + q] *= f;
            mw[n][q] = w - PA_AIM;
          }
        }
    }
    // weights, transposed from [tokens x queries] to the B operand
    uint32_t p[2][NT][2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float w[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            l[n][q] += fast_exp2(s[g][n][2 * i + q] - ms[n][q]);
            w[q] = fast_exp2(x[g][n][2 * i + q] - mw[n][q]);
          }
          const __half2 hv = __floats2half2_rn(w[0], w[1]);
          p[g][n][i] = transpose8x8(*reinterpret_cast<const uint32_t*>(&hv));
        }
    // O^T += V^T P^T: tile j takes this lane's dims 2j and 2j + 1
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t v[4][DH / 32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 16 * g + 8 * (i >> 1) + 2 * c + (i & 1);
        if constexpr (DH == 128) {
          const uint4 x = *reinterpret_cast<const uint4*>(st + R::KV_BYTES + R::at(tok, r));
          v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(st + R::KV_BYTES + R::at(tok, r >> 1) + (r & 1) * 8);
          v[i][0] = x.x, v[i][1] = x.y;
        }
      }
#pragma unroll
      for (int m = 0; m < DH / 32; ++m)
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const uint32_t ab = __byte_perm(v[0][m], v[1][m], o ? 0x7362 : 0x5140);
          const uint32_t cd = __byte_perm(v[2][m], v[3][m], o ? 0x7362 : 0x5140);
          const uint32_t a0 = codes_f16x2<KV, 0>(ab), a1 = codes_f16x2<KV, 1>(ab);
          const uint32_t a2 = codes_f16x2<KV, 0>(cd), a3 = codes_f16x2<KV, 1>(cd);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(acc[n][2 * m + o], a0, a1, a2, a3, p[g][n][0], p[g][n][1]);
        }
    }
    __syncwarp();  // every lane is done with the stage
#pragma unroll
    for (int i = 0; i + 1 < R::STAGES; ++i) scales[i] = scales[i + 1];
    issue(u + R::STAGES * PA_WARPS, stage, pg_next, scales[R::STAGES - 1]);
    pg_next = page_of(u + (R::STAGES + 1) * PA_WARPS);
    stage = stage + 1 == R::STAGES ? 0 : stage + 1;
  }
  cp_wait<0>();
  __syncthreads();

  // merge the warps: [warp][row][DH + 4] floats over the ring, a warp a row
  float* part = reinterpret_cast<float*>(sm);
  constexpr int PITCH = DH + 4;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float x = l[n][q];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      float* row = part + (warp * ROWS + n * 8 + 2 * c + q) * PITCH;
#pragma unroll
      for (int j = 0; j < MT; ++j) {
        row[r * (DH / 8) + 2 * j] = acc[n][j][q];
        row[r * (DH / 8) + 2 * j + 1] = acc[n][j][2 + q];
      }
      if (r == 0) *reinterpret_cast<float4*>(row + DH) = make_float4(ms[n][q], mw[n][q], x, 0.f);
    }
  __syncthreads();
  float* joined = part + PA_WARPS * ROWS * PITCH;  // this block's rows, for the cluster
  for (int rl = warp; rl < ROWS; rl += PA_WARPS) {
    const int row = tile * ROWS + rl;
    if (row >= rows) break;
    const float* x = part + rl * PITCH;
    float4 ml[PA_WARPS];
    float MS = PA_LOW, MW = PA_LOW, L = 0.f, o[DH / 32];
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      ml[w] = *reinterpret_cast<const float4*>(x + w * ROWS * PITCH + DH);
      MS = fmaxf(MS, ml[w].x);
      MW = fmaxf(MW, ml[w].y);
    }
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      L += ml[w].z * fast_exp2(ml[w].x - MS);
      const float f = fast_exp2(ml[w].y - MW);
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) o[i] = fmaf(x[w * ROWS * PITCH + i * 32 + lane], f, o[i]);
    }
    const int token = by.group.div(row), head = h * group + row - token * group;
    const int64_t grow = (int64_t)seq * d.q_len + token;
    if (nsplit == 1) {
      const float f = L == 0.f ? 0.f : fast_exp2(MW - MS) / L;
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) ((__nv_bfloat16*)d.out)[grow * d.ldo + head * DH + i * 32 + lane] = __float2bfloat16(o[i] * f);
    } else if (cluster) {
      float* y = joined + rl * PITCH;
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) y[i * 32 + lane] = o[i];
      if (lane == 0) *reinterpret_cast<float4*>(y + DH) = make_float4(MS, MW, L, 0.f);
    } else {
      const int64_t at = (grow * d.Hq + head) * nsplit + split;
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) d.part_o[at * DH + i * 32 + lane] = o[i];
      if (lane == 0) *reinterpret_cast<float4*>(d.part_ml + at * 4) = make_float4(MS, MW, L, 0.f);
    }
  }
  if (!cluster) return;
  // the cluster's blocks share the rows out and read each other's parts, in their order
  cluster_sync();
  for (int rl = split + nsplit * warp; rl < ROWS; rl += nsplit * PA_WARPS) {
    const int row = tile * ROWS + rl;
    if (row >= rows) break;
    const uint32_t mine = smem_u32(joined + rl * PITCH);
    float4 ml = make_float4(PA_LOW, PA_LOW, 0.f, 0.f);
    if (lane < nsplit) ml = ld_cluster4(mapa_shared(mine + DH * 4, lane));
    const float MS = warp_max(ml.x), MW = warp_max(ml.y);
    const float L = warp_sum(ml.z * fast_exp2(ml.x - MS)), f = fast_exp2(ml.y - MW);
    float o[DH / 32];
#pragma unroll
    for (int i = 0; i < DH / 32; ++i) o[i] = 0.f;
#pragma unroll 4
    for (int q = 0; q < nsplit; ++q) {
      const float g = __shfl_sync(0xffffffffu, f, q);
      const uint32_t there = mapa_shared(mine + lane * 4, q);
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) o[i] = fmaf(ld_cluster(there + i * 128), g, o[i]);
    }
    const int token = by.group.div(row), head = h * group + row - token * group;
    const float g = L == 0.f ? 0.f : fast_exp2(MW - MS) / L;
#pragma unroll
    for (int i = 0; i < DH / 32; ++i)
      ((__nv_bfloat16*)d.out)[((int64_t)seq * d.q_len + token) * d.ldo + head * DH + i * 32 + lane] = __float2bfloat16(o[i] * g);
  }
  cluster_sync();  // no block leaves while another reads its shared memory
}

// Joins the parts of a (row, head), a block each: every warp finds the references and
// the sum from all parts (a lane per part), then takes every fourth part's output, eight
// of them on their way at once.  Sums are in a fixed order.  (A warp alone, part after
// part, took 14 us for 18 parts and 24 us for 37.)
constexpr int JOIN_WARPS = 4;

template <int DH>
__global__ void __launch_bounds__(32 * JOIN_WARPS) page_attn_join_kernel(LkPageAttnDesc d, int tile_rows, int nsplit) {
  __shared__ float so[JOIN_WARPS][DH];
  const int64_t w = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t grow = w / d.Hq;
  const int head = (int)(w % d.Hq), group = d.Hq / d.Hkv;
  const int row = (int)(grow % d.q_len) * group + head % group;
  const int last = min(group * d.q_len, (row / tile_rows + 1) * tile_rows) - 1;
  const PaSpan sp = page_attn_span(d, d.ctx_lens[grow / d.q_len], last / group);
  const int used = max(1, (sp.units + sp.per - 1) / sp.per);
  cudaGridDependencySynchronize();  // the parts are written
  const float4* ml = reinterpret_cast<const float4*>(d.part_ml) + w * nsplit;
  const float* po = d.part_o + w * nsplit * DH + lane;
  float MS = PA_LOW, MW = PA_LOW, L = 0.f, o[DH / 32];
  for (int s = lane; s < used; s += 32) {
    const float4 x = ml[s];
    MS = fmaxf(MS, x.x);
    MW = fmaxf(MW, x.y);
  }
  MS = warp_max(MS);
  MW = warp_max(MW);
#pragma unroll
  for (int i = 0; i < DH / 32; ++i) o[i] = 0.f;
  for (int base = 0; base < used; base += 32) {
    const float4 x = base + lane < used ? ml[base + lane] : make_float4(PA_LOW, PA_LOW, 0.f, 0.f);
    L += x.z * fast_exp2(x.x - MS);
    const float f = base + lane < used ? fast_exp2(x.y - MW) : 0.f;
    float v[32 / JOIN_WARPS][DH / 32];
#pragma unroll
    for (int k = 0; k < 32 / JOIN_WARPS; ++k) {
      const int s = base + warp + JOIN_WARPS * k;
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) v[k][i] = s < used ? po[(int64_t)s * DH + i * 32] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 32 / JOIN_WARPS; ++k) {
      const float g = __shfl_sync(0xffffffffu, f, warp + JOIN_WARPS * k);
#pragma unroll
      for (int i = 0; i < DH / 32; ++i) o[i] = fmaf(v[k][i], g, o[i]);
    }
  }
  L = warp_sum(L);
#pragma unroll
  for (int i = 0; i < DH / 32; ++i) so[warp][i * 32 + lane] = o[i];
  __syncthreads();
  const float f = fast_exp2(MW - MS);
  for (int c = threadIdx.x; c < DH; c += 32 * JOIN_WARPS) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < JOIN_WARPS; ++k) x += so[k][c];
    ((__nv_bfloat16*)d.out)[grow * d.ldo + head * DH + c] = __float2bfloat16(L == 0.f ? 0.f : x * f / L);
  }
}

template <int KV, int DH, int NT>
struct PaKernel {
  static constexpr int merge = (PA_WARPS + 1) * 8 * NT * (DH + 4) * 4, ring = PA_WARPS * PaRing<DH>::WARP;
  static constexpr int smem = ring > merge ? ring : merge;

  static void config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& attr, int64_t blocks, int nsplit) {
    cfg = cudaLaunchConfig_t{};
    attr = cudaLaunchAttribute{};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(32 * PA_WARPS);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    if (nsplit > 1 && nsplit <= PA_CLUSTER) {
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = nsplit;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.numAttrs = 1;
    }
  }

  // Kernel attributes of the current device, set once; and how many blocks it holds at a time
  // when they come in clusters of c (0: singly), which the GPU's partition limits: of 2
  // blocks an SM on 148 SMs 296 singly, 270 by sixes, 224 by sixteens.
  static const int* places() {
    struct Table {
      std::once_flag once;
      int at[PA_CLUSTER + 1] = {0};
    };
    static Table tables[64];
    int dev = 0;
    cudaGetDevice(&dev);
    Table& t = tables[dev & 63];
    std::call_once(t.once, [&] {
      auto k = page_attn_kernel<KV, DH, NT>;
      if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
          cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return;
      int blocks = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, k, 32 * PA_WARPS, smem) != cudaSuccess) return;
      t.at[0] = t.at[1] = blocks * num_sms();
      for (int c = 2; c <= PA_CLUSTER; ++c) {
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr;
        config(cfg, attr, (int64_t)c * num_sms(), c);
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, k, &cfg) == cudaSuccess) t.at[c] = n * c;
      }
      cudaGetLastError();  // a size that does not fit is a 0 here, not an error
    });
    return t.at;
  }

  static int launch(const LkPageAttnDesc& d, cudaStream_t s) {
    const int rows = d.Hq / d.Hkv * d.q_len, tiles = cdiv(rows, 8 * NT);
    const int64_t blocks = (int64_t)d.num_seqs * d.Hkv * tiles * d.nsplit;
    LK_REQUIRE(blocks < (1ll << 31) && (int64_t)d.num_seqs * d.q_len * d.Hq < (1ll << 31),
               "page_attention: too many rows in one call");
    if (places()[0] == 0) return check_launch("page_attention: kernel attributes") ? -1 : fail("page_attention: no room for a block");
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr;
    config(cfg, attr, blocks, d.nsplit);
    cfg.stream = s;
    cudaLaunchKernelEx(&cfg, page_attn_kernel<KV, DH, NT>, d,
                       PaDivs{FastDiv(d.nsplit), FastDiv(d.Hkv), FastDiv(tiles), FastDiv(d.Hq / d.Hkv), FastDiv(d.page)});
    if (check_launch("page_attention")) return -1;
    if (d.nsplit <= PA_CLUSTER) return 0;
    // launched while the parts still run (its blocks wait for them in the launch order of
    // the stream): the launch's own latency is not waited for
    cfg.gridDim = dim3((unsigned)((int64_t)d.num_seqs * d.q_len * d.Hq));
    cfg.blockDim = dim3(32 * JOIN_WARPS);
    cfg.dynamicSmemBytes = 0;
    attr = cudaLaunchAttribute{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, page_attn_join_kernel<DH>, d, 8 * NT, d.nsplit);
    return check_launch("page_attention_join");
  }
};

template <typename F>  // f(PaKernel of these types and sizes)
static auto page_attn_variant(int kv_dtype, int Dh, int64_t rows, F f) {
#define LK_PA(KV, DH) (rows > 8 ? f(PaKernel<KV, DH, 2>()) : f(PaKernel<KV, DH, 1>()))
  if (kv_dtype == 1) return Dh == 64 ? LK_PA(1, 64) : LK_PA(1, 128);
  return Dh == 64 ? LK_PA(2, 64) : LK_PA(2, 128);
#undef LK_PA
}

}  // namespace lk

using namespace lk;

// Into how many parts a context may be cut, from the longest context that the host expects
// (each block cuts its sequence's own length).
// The estimate, in tokens that an SM takes at its full rate (which two blocks reach, one
// 60 % of it): a part and what a block costs beside it (150 tokens: 2.3 us shared by the
// blocks of an SM), in waves of as many blocks as are resident at a time in clusters of
// this size; half of that for equal lengths, half the same work spread evenly for lengths
// that are 0.6 of the longest, but no less than the longest part alone; and 60 more for
// the join of a cluster, 300 for a second launch (more than 16 parts).
// Measured (us on the device, 32 heads on 8 KV heads of 128 where not said: uncut, chosen, the
// best of 1 to 16 parts): 1 x 2000 15.7, 6.4, 6.5; 1 x 30000 257, 19.3 (over 16 parts), 23.7;
// 8 x 4096 36.5, 13.5, 13.4; 16 x 4096 37.3, 21.8, 21.8; 32 x 4096 42.5, 34.9, 34.8; 64 x 4096
// 60.3, 61.2, 58.1; 32 x 500 7.7, 7.7, 7.7; 24 x 2047 (4 heads of 64, int8) 13.9, 10.3, 10.1;
// 24 new tokens over 2000 20.0, 12.7, 12.8 (20.9 in 6 parts, whose clusters need a second wave).
// A batch that fills the GPU by itself is not cut, whatever max_ctx says: in a captured step that
// is the longest context the server allows, not the batch's.  256 sequences of up to 2000 tokens
// take 95 us at any max_ctx; in parts of 4096 they took 157 us for a max_ctx of 8192 and 619 for
// 32768 (the parts' blocks without tokens hold their places until their cluster is done), 157 and
// 237 where such blocks left at once, which is what starting them costs.  Uncut, a long context
// among short ones runs on alone: 30000 tokens beside 255 sequences of up to 500 (2000) take 288
// (336) us, against 358 (640) and 155 (258) in those two forms.
extern "C" int lk_page_attention_splits(int num_seqs, int q_len, int Hq, int Hkv, int Dh, int kv_dtype, int max_ctx) {
  const int64_t rows = (int64_t)(Hq / Hkv) * q_len, blocks = std::max<int64_t>(1, num_seqs * Hkv * (rows <= 8 ? 1 : (rows + 15) / 16));
  const int sms = num_sms(), most = max_ctx <= 256 ? 1 : cdiv(max_ctx, 256);
  const int* places = page_attn_variant(kv_dtype, Dh, rows, [](auto k) { return decltype(k)::places(); });
  const int full = (int)std::min<int64_t>(most, places[0] / blocks + 1), step = std::max(1, full / 32);
  int best = 1;
  double least = 1e30;
  auto wave = [&](double part, double held) {  // blocks of an SM: held
    return part * held / std::min(1.0, 0.6 * held);
  };
  auto consider = [&](int64_t ns) {
    if (ns < 1 || ns > full) return;
    const int64_t all = blocks * ns, room = std::max(1, ns <= PA_CLUSTER ? places[ns] : places[0]) / ns * ns;
    if (room == 0) return;
    const double part = (double)max_ctx / ns + 150;
    const int64_t waves = all / room, rest = all % room;
    const double even = waves * wave(part, (double)room / sms) + (rest ? wave(part, (double)((rest + sms - 1) / sms)) : 0.0);
    const double mixed = num_seqs > 1 ? std::max(0.6 * part * all / sms, part / 0.6) : even;
    const double cost = 0.5 * (even + mixed) + (ns > PA_CLUSTER ? 300 : ns > 1 ? 60 : 0);
    if (cost < least) least = cost, best = (int)ns;
  };
  for (int ns = 1; ns <= std::min(full, PA_CLUSTER); ++ns) consider(ns);
  for (int ns = PA_CLUSTER + 1; ns <= full; ns += step) consider(ns);
  for (int k = 1; k <= 3; ++k) consider((int64_t)k * sms / blocks);
  return best;
}

extern "C" int lk_page_attention(const LkPageAttnDesc* d, cudaStream_t s) {
  LK_REQUIRE(d->Dh == 64 || d->Dh == 128, "page_attention: head_dim must be 64 or 128");
  if (d->num_seqs == 0) return 0;
  LK_REQUIRE(d->nsplit <= PA_CLUSTER || (d->part_o && d->part_ml), "page_attention: split partial buffers needed");
  return page_attn_variant(d->kv_dtype, d->Dh, (int64_t)(d->Hq / d->Hkv) * d->q_len,
                           [&](auto k) { return decltype(k)::launch(*d, s); });
}
