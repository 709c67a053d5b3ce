// Block-scaled 8-bit paged KV cache: write, decode attention (with accumulated attention weights),
// block dequantization, and eviction by accumulated weight.
//
// Layout of one layer: codes [NB, 2, Hk, bs, D] (int8, or e4m3 bit patterns) and one fp32 scale per
// (block, K/V, kv head): scales [NB, 2, Hk]; value = code * scale. bs is 16, 32 or 64. Optional:
// mass [NB, Hk, bs] fp32, the softmax weight each cached token has drawn so far, summed over the
// queries and over the heads of its group.
//
// The scales that are written are powers of two (at least 2^-100), so value / scale and its rounding
// are exact in any precision: a code is a function of the inputs alone, requantizing a block whose
// scale grows is a shift, and the bf16 copy that prompt attention reads holds every value exactly (but for 2^128, what
// the largest bf16's code rounds to, in whose place it holds the largest bf16).
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../common/common.cuh"
#include "../common/tma_host.h"
#include "launchers.h"

namespace gollek {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------------------------------------
// Codes and scales
// ---------------------------------------------------------------------------------------------
// The smallest power of two s with amax <= qmax * s (qmax 127 or 448), at least 2^-100. With
// amax = 1.f * 2^E: s = 2^(E - 6) for int8 unless 1.f > 127/64, 2^(E - 8) for e4m3 unless 1.f > 7/4.
template <bool E4M3>
GOLLEK_DEVICE float pow2_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int E = (int)(b >> 23) - 127;
  const uint32_t mant = b & 0x7fffffu;
  int e = E4M3 ? E - 8 + (mant > 0x600000u) : E - 6 + (mant > 0x7e0000u);
  e = max(e, -100);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// y = value / scale -> code (round to nearest, ties to even, saturating)
template <bool E4M3>
GOLLEK_DEVICE uint32_t encode4(float y0, float y1, float y2, float y3) {
  if constexpr (E4M3) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y2, y3), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  } else {
    auto c = [](float y) { return (uint32_t)(max(-127, min(127, __float2int_rn(y))) & 0xff); };
    return c(y0) | (c(y1) << 8) | (c(y2) << 16) | (c(y3) << 24);
  }
}
template <bool E4M3>
GOLLEK_DEVICE void decode4(uint32_t w, float* f) {
  if constexpr (E4M3) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 fa = __half22float2(*reinterpret_cast<const __half2*>(&a));
    const float2 fb = __half22float2(*reinterpret_cast<const __half2*>(&b));
    f[0] = fa.x, f[1] = fa.y, f[2] = fb.x, f[3] = fb.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  }
}

// ---------------------------------------------------------------------------------------------
// Write: one warp per (run of tokens that share a block, K/V, kv head).
//
// A run is found by its first token: the token whose nearest earlier token with a slot lies in another block.
// The warp takes the run's largest magnitude, fixes the block's scale (a run that writes the block's
// first slot starts the block anew, any other can only raise the scale), rounds the codes already
// there to a raised scale, and stores the run's codes. Memory-bound: 3 bytes a value. A run of at most 16 tokens stays
// in registers between its magnitude and its codes (16-byte loads, all of them in flight at once); a longer one is read twice.
// Measured (8 heads of 128): 48 rows of one token 3.2 us, the latency of slot, first code and scale one behind the other (4.1 to
// 4.8 us where every scale grows); 8190 prompt tokens in blocks of 16 14.6 us, 3.4 TB/s: bytes in flight, with the 20 warps an SM
// holds at 96 registers (16 at 126: 16.4 us; 24 at 80 spill: 18 us). A run that does not stay in registers is stored a token at
// a time, behind the load of its slot: in blocks of 32 and 64, whose runs are longer, the same tokens take 45 and 49 us. So are
// the runs of a prompt whose first tokens are the last of their warps' 16 (lane 16), for the next block's first token is not seen: 38
// us behind 15 decode rows. And in a step of 1024 tokens a warp takes up to 16 decode rows one behind the other: a prompt behind
// 16 to 256 of them takes 30 us.
// ---------------------------------------------------------------------------------------------
GOLLEK_DEVICE uint32_t clean2(uint32_t w) {  // two bf16: NaN -> 0, infinities -> the largest bf16
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 32; i += 16) {
    const uint32_t x = (w >> i) & 0xffffu, a = x & 0x7fffu;
    r |= (a > 0x7f80u ? 0u : a == 0x7f80u ? (x & 0x8000u) | 0x7f7fu : x) << i;
  }
  return r;
}
GOLLEK_DEVICE uint4 clean8(const uint4& u) { return make_uint4(clean2(u.x), clean2(u.y), clean2(u.z), clean2(u.w)); }
// Running maximum of magnitudes in two bf16 lanes (NaN stays visible).
GOLLEK_DEVICE void top8(uint32_t& m, const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = w[i] & 0x7fff7fffu;
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(a));
  }
}
GOLLEK_DEVICE bool not_finite(uint32_t m) { return (m & 0x7fffu) >= 0x7f80u || (m >> 16) >= 0x7f80u; }
GOLLEK_DEVICE float top_value(uint32_t m) { return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)); }
// Eight bf16 times inv -> codes; |value * inv| <= qmax and the product is exact, so adding 1.5 * 2^23 rounds it to the
// integer (ties to even) that the sum's low byte is.
template <bool E4M3>
GOLLEK_DEVICE uint2 encode8(const uint4& u, float inv) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t c[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float a = __uint_as_float(w[2 * i] << 16), b = __uint_as_float(w[2 * i] & 0xffff0000u);
    const float d = __uint_as_float(w[2 * i + 1] << 16), e = __uint_as_float(w[2 * i + 1] & 0xffff0000u);
    if constexpr (E4M3) {
      c[i] = encode4<true>(a * inv, b * inv, d * inv, e * inv);
    } else {
      constexpr float kRound = 12582912.f;
      const uint32_t x = __byte_perm(__float_as_uint(fmaf(a, inv, kRound)), __float_as_uint(fmaf(b, inv, kRound)), 0x0040);
      const uint32_t y = __byte_perm(__float_as_uint(fmaf(d, inv, kRound)), __float_as_uint(fmaf(e, inv, kRound)), 0x0040);
      c[i] = __byte_perm(x, y, 0x5410);
    }
  }
  return make_uint2(c[0], c[1]);
}

// Two bf16: infinities -> the largest bf16 (NaN stays). Its code rounds up to 2^128, so a value read back may pass fp32's range.
GOLLEK_DEVICE uint32_t saturate2(uint32_t w) {
  asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0x7f7f7f7fu));
  asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0xff7fff7fu));
  return w;
}

struct QuantArgs {
  const __nv_bfloat16* kv;
  int64_t st, sw, sh;  // element strides of kv [T, 2, Hk, D]
  const int* slots;
  uint8_t* cache;
  float* scales;
  float* mass;
  int T, Hk, bs_log2, num_blocks, g;  // g: tokens a warp looks at
  uint32_t* bounds;
};

constexpr int kQuantThreads = 128;

template <bool E4M3, int D>
__global__ void __launch_bounds__(kQuantThreads, D <= 64 ? 6 : D <= 128 ? 5 : 3) kv_quant_blocks_kernel(const QuantArgs p) {
  constexpr int LPR = D / 8, TPI = 32 / LPR;      // lanes of a row (8 values each), rows a warp takes at once
  constexpr int R = (16 + TPI - 1) / TPI;         // rounds for 16 rows
  const int64_t gw = (int64_t)blockIdx.x * (kQuantThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, sub = lane / LPR, pos = lane % LPR;
  const int64_t grp = gw / (2 * p.Hk);
  const int pair = (int)(gw - grp * (2 * p.Hk));
  const int t0 = (int)(grp * p.g);
  if (t0 >= p.T) return;
  const int w = pair / p.Hk, h = pair - w * p.Hk;
  const int bs = 1 << p.bs_log2;
  const __nv_bfloat16* kv = p.kv + w * p.sw + h * p.sh + pos * 8;
  // lane i: slot of token t0 - 1 + i; lanes 1 .. g are this warp's tokens, the others show where a run ends
  const int tl = t0 - 1 + lane;
  const int sl = tl >= 0 && tl < p.T ? p.slots[tl] : -1;
  const int bl = sl >= 0 ? sl >> p.bs_log2 : -1;
  const int bp = __shfl_up_sync(0xffffffffu, bl, 1);
  uint32_t leaders = __ballot_sync(0xffffffffu, lane >= 1 && lane <= p.g && bl >= 0 && bl != bp);
  while (leaders) {
    const int li = __ffs(leaders) - 1;
    leaders &= leaders - 1;
    const int tlead = t0 - 1 + li;
    const int blk = __shfl_sync(0xffffffffu, bl, li);
    if (__shfl_sync(0xffffffffu, bp, li) < 0) {  // a skipped token (or none) before it: look for the nearest one with a slot
      int back = tlead - 1;
      while (back >= 0 && p.slots[back] < 0) --back;
      if (back >= 0 && (p.slots[back] >> p.bs_log2) == blk) continue;
    }
    if (checked_index(blk, p.num_blocks, p.bounds, -1) < 0) continue;  // beyond the pool (where bounds are checked): skipped
    const int64_t row = ((int64_t)blk * 2 + w) * p.Hk + h;
    uint8_t* codes = p.cache + (row << p.bs_log2) * D;
    // the run's tokens among the lanes, and whether they are all of it
    const uint32_t other = __ballot_sync(0xffffffffu, lane > li && bl >= 0 && bl != blk);
    const uint32_t run = __ballot_sync(0xffffffffu, lane >= li && bl >= 0 && (other == 0 || lane < __ffs(other) - 1));
    const int span = 32 - __clz(run) - li;  // tokens from the first to the last one
    const int off = bl == blk && ((run >> lane) & 1) ? sl & (bs - 1) : 64;
    uint64_t written = (uint64_t)__reduce_or_sync(0xffffffffu, off < 32 ? 1u << off : 0u) |
                       ((uint64_t)__reduce_or_sync(0xffffffffu, off >= 32 && off < 64 ? 1u << (off - 32) : 0u) << 32);
    const bool held = (other != 0 || tlead - li + 32 >= p.T) && span <= 16 && __popc(run) == __popcll(written);
    uint4 raw[R];
    uint32_t m = 0;
    bool special = false;
    int tend = tlead;
    if (held) {  // at most 16 tokens, every slot once: they stay in registers
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = r * TPI + sub;
        raw[r] = make_uint4(0u, 0u, 0u, 0u);
        if (sub < TPI && i < span && ((run >> (li + i)) & 1)) raw[r] = *reinterpret_cast<const uint4*>(kv + (int64_t)(tlead + i) * p.st);
      }
    } else {
      written = 0;
      for (bool more = true; more && tend < p.T;) {
        const int s = tend + lane < p.T ? p.slots[tend + lane] : -1;
        const uint32_t om = __ballot_sync(0xffffffffu, s >= 0 && (s >> p.bs_log2) != blk);
        const int n = min(p.T - tend, om ? __ffs(om) - 1 : 32);
        more = om == 0;
        for (int i0 = 0; i0 < n; i0 += 16) {
          bool bad = false;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const int i = i0 + r * TPI + sub;
            const int si = __shfl_sync(0xffffffffu, s, i & 31);
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (sub < TPI && i < min(n, i0 + 16) && si >= 0) u = *reinterpret_cast<const uint4*>(kv + (int64_t)(tend + i) * p.st);
            uint32_t x = 0;
            top8(x, u);
            if (not_finite(x)) {
              bad = true;
              x = 0;
              top8(x, clean8(u));
            }
            asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(x));
          }
          special |= bad;
        }
        const int o = s >= 0 && lane < n ? s & (bs - 1) : 64;
        written |= (uint64_t)__reduce_or_sync(0xffffffffu, o < 32 ? 1u << o : 0u) |
                   ((uint64_t)__reduce_or_sync(0xffffffffu, o >= 32 && o < 64 ? 1u << (o - 32) : 0u) << 32);
        tend += n;
      }
    }
    const float old = p.scales[row];
    if (held) {
#pragma unroll
      for (int r = 0; r < R; ++r) top8(m, raw[r]);
      if (not_finite(m)) {
        m = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          raw[r] = clean8(raw[r]);
          top8(m, raw[r]);
        }
      }
    }
    const float need = pow2_scale<E4M3>(warp_max(top_value(m)));
    const bool fresh = written & 1;
    const float s = fresh ? need : fmaxf(old, need);
    if (!fresh && s > old) {  // the block's scale grows: round what it holds to the new one
      const float ratio = old / s;
#pragma unroll 1
      for (int o0 = 0; o0 < bs; o0 += R * TPI) {
        uint2 c[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int o = o0 + r * TPI + sub;
          if (sub < TPI && o < bs) c[r] = *reinterpret_cast<const uint2*>(codes + o * D + pos * 8);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int o = o0 + r * TPI + sub;
          if (sub >= TPI || o >= bs || ((written >> o) & 1)) continue;
          float f[8];
          decode4<E4M3>(c[r].x, f);
          decode4<E4M3>(c[r].y, f + 4);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= ratio;
          *reinterpret_cast<uint2*>(codes + o * D + pos * 8) =
              make_uint2(encode4<E4M3>(f[0], f[1], f[2], f[3]), encode4<E4M3>(f[4], f[5], f[6], f[7]));
        }
      }
    }
    __syncwarp();
    if (lane == 0) p.scales[row] = s;
    const float inv = 1.f / s;
    const bool mass = p.mass != nullptr && w == 0 && pos == 0;
    float* ms = p.mass + (((int64_t)blk * p.Hk + h) << p.bs_log2);
    if (held) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int i = r * TPI + sub, o = __shfl_sync(0xffffffffu, off, (li + i) & 31);
        if (sub >= TPI || i >= span || !((run >> (li + i)) & 1)) continue;
        *reinterpret_cast<uint2*>(codes + o * D + pos * 8) = encode8<E4M3>(raw[r], inv);
        if (mass) ms[o] = 0.f;
      }
    } else {  // tokens in order: of two with the same slot the later one stays
      special = __any_sync(0xffffffffu, special);
      for (int t = tlead; t < tend; ++t) {
        const int slot = p.slots[t];
        if (slot < 0 || sub != 0) continue;
        const int o = slot & (bs - 1);
        uint4 u = *reinterpret_cast<const uint4*>(kv + (int64_t)t * p.st);
        if (special) u = clean8(u);
        *reinterpret_cast<uint2*>(codes + o * D + pos * 8) = encode8<E4M3>(u, inv);
        if (mass) ms[o] = 0.f;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// bf16 copy of the listed blocks (exact: an 8-bit code times a power of two), for prompt attention:
// in blocks of 16 tokens whatever the cache's block size, [rows * mb16, 2, Hk, 16, D], or with a sequence's
// tokens of a head together, [rows, 2, Hk, mb16 * 16, D] (a KV tile is then one box). Row r of
// the table holds lens[r] tokens: what lies behind them reads as zero up to the next multiple
// of 128 tokens (the prompt kernels' KV tile) and is not written beyond it. 8 codes a lane: a warp stores 512 bytes on end.
// Memory-bound, 3 bytes a value: 48k tokens of 8 heads of 64 in 26 us, 5.6 TB/s (four CTAs an SM; three, with twice the loads
// of a thread in flight, 29 us; 16 codes a lane, whose stores fill half a sector each, 31 us).
// ---------------------------------------------------------------------------------------------
template <bool E4M3, int D>
__global__ void __launch_bounds__(256, 4)
    kv_dequant_scaled_kernel(const uint8_t* __restrict__ cache, const float* __restrict__ scales,
                             const int* __restrict__ tables, int64_t bt_stride, const int* __restrict__ lens, int mb16,
                             int width, int num_blocks, int Hk, int bs_log2, __nv_bfloat16* __restrict__ dst,
                             const PromptRows prompt, uint32_t* bounds) {
  const int r = blockIdx.y, i = blockIdx.x;             // table row, 16-token block of the row
  const int L = lens ? min(max(lens[r], 0), width) : width;
  if (prompt.lens != nullptr) {
    if (prompt.ids != nullptr && threadIdx.x == 0) prompt.ids[(int64_t)r * mb16 + i] = r * mb16 + i;
    if (i == 0) {
      if (threadIdx.x == 0) prompt.lens[r] = L;
      const int q0 = prompt.query_start[r], none = prompt.query_start[r + 1] - q0 - L;
      for (int t = 0; t < none; ++t)
        for (int x = threadIdx.x * 8; x < prompt.width; x += 256 * 8)
          *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(prompt.out) + (q0 + t) * prompt.out_stride + x) =
              make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const int tok0 = i << 4;
  constexpr int vec = D / 8;                            // 8-code vectors per token row
  const int n = tok0 < ((L + 127) & ~127) ? 2 * Hk * vec << 4 : 0;  // of the destination block
  int64_t id = 0;
  if (tok0 < L) id = checked_index(tables[(int64_t)r * bt_stride + (tok0 >> bs_log2)], num_blocks, bounds);
  const int off0 = tok0 & ((1 << bs_log2) - 1);
  // first row of (K/V, head) 0, and the distance of the next one
  const int64_t row0 = prompt.together ? (int64_t)r * 2 * Hk * mb16 * 16 + tok0 : ((int64_t)r * mb16 + i) * 2 * Hk * 16;
  const int64_t hrow = prompt.together ? (int64_t)mb16 * 16 : 16;
  constexpr int N = 4;                                  // loads of a thread in flight
  for (int v0 = threadIdx.x; v0 < n; v0 += N * 256) {
    uint2 c[N];
    float s[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int v = v0 + k * 256, rowi = v / vec;       // (K/V, head, token)
      c[k] = make_uint2(0u, 0u);
      s[k] = 0.f;
      if (v < n && tok0 + (rowi & 15) < L) {
        const int64_t row = id * 2 * Hk + (rowi >> 4);
        s[k] = scales[row];
        c[k] = reinterpret_cast<const uint2*>(cache)[((row << bs_log2) + off0 + (rowi & 15)) * vec + v % vec];
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int v = v0 + k * 256;
      if (v >= n) break;
      float f[8];
      decode4<E4M3>(c[k].x, f);
      decode4<E4M3>(c[k].y, f + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= s[k];
      const int rowi = v / vec;
      uint4 u = float_to_bf16x8(f);
      u = make_uint4(saturate2(u.x), saturate2(u.y), saturate2(u.z), saturate2(u.w));  // an infinity would reach masked queries
      reinterpret_cast<uint4*>(dst)[(row0 + (rowi >> 4) * hrow + (rowi & 15)) * vec + v % vec] = u;
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched beside the plan: it is done when this kernel is
}

// ---------------------------------------------------------------------------------------------
// Decode attention.
//
// The work is cut into steps of T tokens of one (sequence, kv head, head tile); all steps of the
// batch form one list (sequence by sequence) and every CTA of a grid that just fills the GPU takes an
// equal stretch of it, whatever the lengths: no tail, one prologue per CTA, and loads that run ahead over the
// borders of sequences. A stretch's first and last sequence may be shared with its neighbours: their partial sums
// meet in a second kernel (block8_join_kernel).
//
// A step: warp w (of W) takes the scores of its 16 tokens, S^T = K Q^T, then all warps exchange the
// probabilities in shared memory and warp w takes dims [w D / W, (w + 1) D / W) of O^T = V^T P^T over all T
// tokens, so O is never reduced across warps. Heads are the N = 8 columns of mma.m16n8k16, tokens and
// dims its 16 rows: a group of up to 8 heads wastes no row.
//   K, int8: the codes are the operand as they lie (m16n8k32 s8). Q is written to 2^-22 of its head's largest value as
//      three signed digits to the base 256, whose products add up in 32-bit integers. Against codes turned into f16:
//      16 rows of 32k, 64 heads: 174 us, not 193, where the power cap holds the clock.
//   K, e4m3: a lane's four consecutive bytes of a 16-byte chunk become two f16 k-pairs, exactly. Any order of dims will
//      do as long as Q follows it, so Q is gathered in that order once per sequence. (Two e4m3 planes of Q would do for
//      the codes as they lie, but 64 rows of up to 4k took 65.6 us with them, not 61.4.)
//   V: ldmatrix.trans moves byte pairs; a byte permute splits them into f16 fragments (exact) of the even and the odd dims.
// Scores get the key scale, probabilities the value scale. The running reference m of the softmax
// covers score + exponent of the value scale, so p * scale fits f16 whatever the scales; the sum l
// uses p alone. m only moves when a score passes it by 2^8: the vote rides on the barrier that the
// exchange needs anyway.
// Measured: 16 rows of 32k (64 heads, 8 KV heads of 128, int8; 1.07 GB) 167 us, 6.4 TB/s: the bytes. 64 rows of up to 4k (32
// heads, e4m3; 329 MB) 61 us, 5.4 TB/s: 8 us of start, joins and end beside the bytes. One row of 1000 tokens 8.4 us: the
// latency of two launches, block ids, codes and a join. Smaller heads lie further from their bytes, for scores, votes and
// barriers are per token: 64 rows of up to 4k take 51 us at head size 64 (bytes: 29 us) and 42 us at 32 (15 us).
// ---------------------------------------------------------------------------------------------
constexpr float kSlack = 8.f;  // p * scale <= 2^9: within f16

template <int D, int NT>
struct DecShape {
  static constexpr int kChunks = D / 16;                            // 16-byte chunks of a token row
  static constexpr int kWarps = D >= 128 ? 4 : D / 16;              // a warp owns D / (16 W) chunks of O
  static constexpr int kTiles = D == 128 || D == 64 ? 2 : 1;                   // tiles of 16 tokens a warp scores in a step
  static constexpr int kTokens = 16 * kWarps * kTiles;              // of a step
  static constexpr int kOwn = kChunks / kWarps;                     // chunks of O a warp owns
  static constexpr bool kSwizzle = kChunks % 8 == 0;
  // rows of 8 chunks are swizzled, others padded to an odd number: 8 rows of one chunk hit 8 bank groups
  static constexpr int kRow = kSwizzle ? D : (kChunks | 1) * 16;
  static constexpr int kSide = kTokens * kRow;                      // K (or V) of a step
  static constexpr int kQRow = 2 * D + 16;
  static constexpr bool kStageQ = NT == 1;                          // a head tile's Q arrives with its first step
  static constexpr int kQ = kStageQ ? 8 * kQRow : 0;                // (two column tiles leave no room for it)
  static constexpr int kStage = (2 * kSide + kQ + 8 * kWarps * kTiles + 15) / 16 * 16;  // K, V, Q, tile scales
  static constexpr int kStages = D < 64 ? 4 : D == 96 ? 3 : 2;
  static constexpr int kPRow = 2 * kTokens + 16;
  static constexpr int kP = NT * 8 * kPRow;
  static constexpr int kSmem = kStages * kStage + kP;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kFit = (227 * 1024) / (kSmem + 1024 + 2 * kWarps * NT * 8 * 4);
  static constexpr int kRegs = 65536 / (kThreads * (NT == 2 ? (D >= 128 ? 224 : 128) : D >= 128 ? 168 : D == 64 ? 128 : 96));
  static constexpr int kCtas = kFit < kRegs ? kFit : kRegs;         // resident CTAs per SM
};

struct DecArgs {
  const __nv_bfloat16* q;
  const uint8_t* cache;
  const float* scales;
  const int* tables;
  const int* lens;
  __nv_bfloat16* out;
  float* part_o;       // [grid, 2, HB, D]: sums of a stretch's first and last sequence, where it is shared
  float* part_ml;      // [grid, 2, HB, 2]: their reference (log2) and sum of probabilities
  float* row_ml;       // [B * H, 2]: reference and sum of the sequences that one CTA finished (mass)
  int* splits;         // [grid, 4]: the head tile that leaves a CTA's stretch at its end: row (-1: none), tile, first part, parts
  int* spans;          // [B * Hk * NG, 2]: first part and number of parts of each head tile (1: finished) (mass)
  float* scores;       // [B * Hk, mb * bs, G] log2 scores (mass)
  float* mass;
  int64_t q_stride, bt_stride;
  int B, H, Hk, G, NG, grid, mb, bs_log2, num_blocks, window;
  float scale_log2, cap, cap_log2;  // softcap (0: none): 2 / softcap, softcap * log2(e)
  uint32_t* bounds;
};

// 16 bytes global -> shared at constant offsets from both addresses; `bytes` 0 writes zeros instead
template <int DST, int SRC>
GOLLEK_DEVICE void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %2], [%1 + %3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
}
template <int DST, int SRC>
GOLLEK_DEVICE void cp_async16_or_zero(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes), "n"(DST), "n"(SRC)
               : "memory");
}
GOLLEK_DEVICE void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
GOLLEK_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
GOLLEK_DEVICE void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
GOLLEK_DEVICE void ldsm4(uint32_t* r, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
GOLLEK_DEVICE void ldsm4_t(uint32_t* r, uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
GOLLEK_DEVICE uint32_t movm_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
GOLLEK_DEVICE void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
GOLLEK_DEVICE void mma_s8(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
GOLLEK_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^(2 x), below fp32's normal numbers too: beside value scales of 2^122 a weight of 2^-20 is a probability of 2^-142
GOLLEK_DEVICE float ex2_twice(float x) {
  const float y = ex2(x);
  return y * y;
}
// l * 2^d in two steps: l reaches 2^108 beside value scales of 2^-100, where 2^d alone would underflow
GOLLEK_DEVICE float shift_sum(float l, float d) {
  const float h = ex2(0.5f * d);
  return l * h * h;
}
GOLLEK_DEVICE uint32_t hsub2u(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Four codes -> two f16 pairs: bytes (0, 1) and (2, 3), or with SPLIT (0, 2) and (1, 3). int8: byte ^ 0x80 under
// the exponent of 1024 is 1024 + 128 + code; the subtraction of 1152 is exact.
template <bool E4M3, bool SPLIT>
GOLLEK_DEVICE void expand4(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (E4M3) {
    if constexpr (SPLIT) w = __byte_perm(w, 0u, 0x3120);
    const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const __half2_raw y = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    a = *reinterpret_cast<const uint32_t*>(&x);
    b = *reinterpret_cast<const uint32_t*>(&y);
  } else {
    const uint32_t u = w ^ 0x80808080u;
    a = hsub2u(__byte_perm(u, 0x64646464u, SPLIT ? 0x4240 : 0x4140), 0x64806480u);
    b = hsub2u(__byte_perm(u, 0x64646464u, SPLIT ? 0x4341 : 0x4342), 0x64806480u);
  }
}

// Tokens of row b that are attended: [lo, L), in steps of T from the tile that holds lo.
struct DecRow {
  int L, lo, t0, n;
};
GOLLEK_DEVICE DecRow dec_row(const DecArgs& p, int b, int T) {
  DecRow r;
  r.L = min(max(p.lens[b], 0), p.mb << p.bs_log2);
  r.lo = p.window > 0 ? max(0, r.L - p.window) : 0;
  r.t0 = r.lo & ~15;
  r.n = (r.L - r.t0 + T - 1) / T;
  return r;
}
// First step of CTA c's stretch, and the CTA whose stretch holds step x. No stretch is empty: with fewer steps
// than CTAs, the last CTAs take no part (grid is then the number of steps).
GOLLEK_DEVICE int stretch_grid(const DecArgs& p, int64_t total) { return (int)min((int64_t)p.grid, total); }
GOLLEK_DEVICE int64_t stretch_begin(int64_t c, int64_t total, int grid) { return c * total / grid; }
GOLLEK_DEVICE int64_t stretch_of(int64_t x, int64_t total, int grid) { return ((x + 1) * grid - 1) / total; }

// Rows as one list, row b with n(b) * X places: every lane sums the places of an equal range of rows. For whole warps.
template <class N>
struct RowList {
  int B, X, per;
  int64_t mine = 0, upto, total;  // places of this lane's range, and up to its end
  N n;
  GOLLEK_DEVICE RowList(int B, int X, N n) : B(B), X(X), n(n) {
    const int lane = threadIdx.x & 31;
    per = (B + 31) / 32;
    const int r0 = min(B, lane * per), r1 = min(B, r0 + per);
#pragma unroll 8
    for (int i = r0; i < r1; ++i) mine += n(i);
    mine *= X;
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    total = __shfl_sync(0xffffffffu, upto, 31);
  }
  // The row that place x < total lies in; x becomes its place in that row. First the range, then the row in it.
  GOLLEK_DEVICE int find(int64_t& x) const {
    const int lane = threadIdx.x & 31;
    const int range = __ffs(__ballot_sync(0xffffffffu, upto > x)) - 1;
    int64_t before = __shfl_sync(0xffffffffu, upto - mine, range);
    for (int b0 = range * per;; b0 += 32) {
      const int k = b0 + lane < B ? n(b0 + lane) : 0;
      int sum = k;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, k > 0 && before + (int64_t)sum * X > x);
      if (hit) {
        const int li = __ffs(hit) - 1;
        x -= before + (int64_t)__shfl_sync(0xffffffffu, sum - k, li) * X;
        return b0 + li;
      }
      before += (int64_t)__shfl_sync(0xffffffffu, sum, 31) * X;
    }
  }
};

// A place in the list of steps: step s of head tile hg of KV head kh of row b.
struct DecPlace {
  int b, kh, hg, s;
  DecRow r;
};
GOLLEK_DEVICE void next_head(DecPlace& q, const DecArgs& p, int T) {
  q.s = 0;
  if (++q.hg < p.NG) return;
  q.hg = 0;
  if (++q.kh < p.Hk) return;
  q.kh = 0;
  do {
    ++q.b;
    if (q.b < p.B) q.r = dec_row(p, q.b, T);
  } while (q.b < p.B && q.r.n == 0);
}

template <int D, int NT, bool E4M3, bool MASS>
__global__ void __launch_bounds__(DecShape<D, NT>::kThreads, DecShape<D, NT>::kCtas)
    block8_decode_kernel(const DecArgs p) {
  using S = DecShape<D, NT>;
  constexpr int CH = S::kChunks, HB = 8 * NT, W = S::kWarps, TW = S::kTiles, T = S::kTokens, OWN = S::kOwn;
  extern __shared__ __align__(128) uint8_t dsm[];
  __shared__ float sm_x[W][HB], sm_l[W][HB];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int X = p.Hk * p.NG;
  const uint32_t ring = smem_u32(dsm), psm = ring + S::kStages * S::kStage;

  asm volatile("griddepcontrol.launch_dependents;");
  if (threadIdx.x == 0) p.splits[blockIdx.x * 4] = -1;
  // rows without tokens are shared out too
  for (int b = blockIdx.x; b < p.B; b += p.grid)
    if (p.lens[b] <= 0 || p.mb == 0)
      for (int i = threadIdx.x; i < p.H * D / 2; i += S::kThreads) reinterpret_cast<uint32_t*>(p.out + (int64_t)b * p.H * D)[i] = 0u;
  // this CTA's stretch of the list
  auto row_steps = [&](int b) { return dec_row(p, b, T).n; };
  const RowList<decltype(row_steps)> list(p.B, X, row_steps);
  const int64_t total = list.total;
  const int grid = stretch_grid(p, total);
  if ((int)blockIdx.x >= grid) return;
  const int64_t first = stretch_begin(blockIdx.x, total, grid);
  const int count = (int)(stretch_begin(blockIdx.x + 1, total, grid) - first);
  DecPlace at;  // of the next step to issue
  {
    int64_t place = first;
    at.b = list.find(place);
    at.r = dec_row(p, at.b, T);
    const int x = (int)(place / at.r.n);
    at.kh = x / p.NG, at.hg = x % p.NG;
    at.s = (int)(place % at.r.n);
  }

  // block ids of this warp's tiles are read 32 at a time, one batch ahead of their use
  constexpr int BATCH = 32 / TW;  // steps
  DecPlace ahead = at;
  auto load_ids = [&]() {
    int id = 0;
    if (ahead.b < p.B) {
      const int t = ahead.r.t0 + (ahead.s + lane / TW) * T + (warp * TW + lane % TW) * 16;
      if (t < ahead.r.L)
        id = checked_index(p.tables[(int64_t)ahead.b * p.bt_stride + (t >> p.bs_log2)], p.num_blocks, p.bounds);
      ahead.s += BATCH;
      if (ahead.s >= ahead.r.n) next_head(ahead, p, T);
    }
    return id;
  };
  int ids = 0, ids_next = load_ids(), batch = BATCH;
  int issued = 0;
  // a lane's pieces of a tile: 16 bytes at lane * 16 + 512 i, i.e. row lane / CH + 32 / CH i where CH divides 32
  const uint32_t block_bytes = (uint32_t)(2 * p.Hk << p.bs_log2) * D, v_bytes = block_bytes >> 1;
  uint32_t st_issue = ring;  // stage of the next step to issue
  auto issue = [&]() {
    if (issued < count) {
      if (batch == BATCH) ids = ids_next, ids_next = load_ids(), batch = 0;
      const uint32_t st = st_issue, tail = st + 2 * S::kSide + S::kQ;
#pragma unroll
      for (int q = 0; q < TW; ++q) {
        const uint32_t id = __shfl_sync(0xffffffffu, ids, batch * TW + q);
        const int tile = warp * TW + q, t = at.r.t0 + at.s * T + tile * 16;
        const int off = t & ((1 << p.bs_log2) - 1);
        const uint8_t* gk = p.cache + (uint64_t)id * block_bytes + (uint32_t)((at.kh << p.bs_log2) + off) * D;
        const uint8_t* gv = gk + v_bytes;
        if (32 % CH == 0 && t >= at.r.lo && t + 16 <= at.r.L) {  // a whole tile
          constexpr int R = 32 / CH;  // rows per round
          const int row = lane / CH, ch = lane % CH;
          const uint8_t *ck = gk + lane * 16, *cv = gv + lane * 16;
          // with the swizzle a lane's chunk changes with the rounds' row parity bits only
          const uint32_t d0 = st + (tile * 16 + row) * S::kRow + ((S::kSwizzle ? ch ^ (row & 7) : ch) << 4);
          const uint32_t d1 = st + (tile * 16 + row) * S::kRow + ((S::kSwizzle ? ch ^ ((row + R) & 7) : ch) << 4);
          constexpr int N = CH / 2, RB = R * S::kRow;
#define GOLLEK_TILE(I)                                                       \
    if constexpr (I < N) {                                                     \
      cp_async16<(I) * RB, (I) * 512>(((I) & 1) ? d1 : d0, ck);                \
      cp_async16<(I) * RB + S::kSide, (I) * 512>(((I) & 1) ? d1 : d0, cv);     \
    }
          if constexpr (N <= 4) {
            GOLLEK_TILE(0) GOLLEK_TILE(1) GOLLEK_TILE(2) GOLLEK_TILE(3)
          } else {  // D = 256: two rows a round, four different chunks
            const uint32_t d2 = st + (tile * 16 + row) * S::kRow + ((ch ^ ((row + 2 * R) & 7)) << 4);
            const uint32_t d3 = st + (tile * 16 + row) * S::kRow + ((ch ^ ((row + 3 * R) & 7)) << 4);
            GOLLEK_TILE(0) GOLLEK_TILE(1) GOLLEK_TILE(4) GOLLEK_TILE(5)
            cp_async16<2 * RB, 2 * 512>(d2, ck);
            cp_async16<2 * RB + S::kSide, 2 * 512>(d2, cv);
            cp_async16<6 * RB, 6 * 512>(d2, ck);
            cp_async16<6 * RB + S::kSide, 6 * 512>(d2, cv);
            cp_async16<3 * RB, 3 * 512>(d3, ck);
            cp_async16<3 * RB + S::kSide, 3 * 512>(d3, cv);
            cp_async16<7 * RB, 7 * 512>(d3, ck);
            cp_async16<7 * RB + S::kSide, 7 * 512>(d3, cv);
          }
#undef GOLLEK_TILE
        } else {
#pragma unroll 1
          for (int i = 0; i < CH / 2; ++i) {
            const int e = i * 32 + lane, row = e / CH, ch = e % CH;
            const int bytes = t + row >= at.r.lo && t + row < at.r.L ? 16 : 0;  // rows outside read as zero
            const uint32_t d = st + (tile * 16 + row) * S::kRow + ((S::kSwizzle ? ch ^ (row & 7) : ch) << 4);
            cp_async16_or_zero<0, 0>(d, gk + e * 16, bytes);
            cp_async16_or_zero<S::kSide, 0>(d, gv + e * 16, bytes);
          }
        }
        if (lane < 2) cp_async4(tail + 8 * tile + 4 * lane, p.scales + (uint64_t)(id * 2 + lane) * p.Hk + at.kh);
      }
      if (S::kStageQ && (at.s == 0 || issued == 0)) {
        const int h0 = at.hg * HB, nh = min(p.G - h0, HB);
        const __nv_bfloat16* q = p.q + (int64_t)at.b * p.q_stride + (int64_t)(at.kh * p.G + h0) * D;
        for (int e = threadIdx.x; e < HB * D / 8; e += S::kThreads) {
          const int hh = e / (D / 8);
          cp_async16_or_zero<0, 0>(st + 2 * S::kSide + hh * S::kQRow + (e % (D / 8)) * 16, hh < nh ? q + e * 8 : q, hh < nh ? 16 : 0);
        }
      }
      ++issued;
      ++batch;
      st_issue = st_issue == ring + (S::kStages - 1) * S::kStage ? ring : st_issue + S::kStage;
      if (++at.s == at.r.n) {
        next_head(at, p, T);
        batch = BATCH;
      }
    }
    cp_async_commit();
  };
  DecPlace cur = at;  // the step being computed
#pragma unroll
  for (int j = 0; j < S::kStages - 1; ++j) issue();

  constexpr int PL = E4M3 ? 2 : 3;  // registers of Q a chunk of 16 dims: two f16 pairs, or three digits
  uint32_t qf[NT][CH][PL];
  float qmul[NT][2];
  float o[OWN][NT][4];
  float m[NT][2], l[NT][2];
  const int frow = (lane & 7) + ((lane >> 3) & 1) * 8, fhi = lane >> 4;  // this lane's row and chunk of an x4 ldmatrix
  bool begun = false;  // whether this stretch holds the current head tile's first step
  uint32_t st = ring;
  for (int j = 0; j < count; ++j) {
    cp_async_wait<S::kStages - 2>();
    __syncthreads();  // the step's data is there, and the previous one's stage is free
    issue();
    const uint32_t tail = st + 2 * S::kSide + S::kQ;
    const int b = cur.b, kh = cur.kh, h0 = cur.hg * HB, nh = min(p.G - h0, HB);
    const int tok0 = cur.r.t0 + cur.s * T;
    if (cur.s == 0 || j == 0) {
      begun = cur.s == 0;
      // Q^T as the B operand, columns = heads: dims 16 i + 4 c + {0 .. 3} of the lane's head. A power of two brings the
      // head's amax to [2^11, 2^12), where f16 holds every bf16 within 2^-28 of it exactly, or to [2^21, 2^22).
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint2 raw[CH];
        float amax = 0.f, poison = 0.f;  // NaN where the head holds a NaN or an infinity
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          if constexpr (S::kStageQ) {
            asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];"
                         : "=r"(raw[i].x), "=r"(raw[i].y)
                         : "r"(st + 2 * S::kSide + (nt * 8 + g) * S::kQRow + 32 * i + 8 * c)
                         : "memory");
          } else {
            raw[i] = make_uint2(0u, 0u);
            if (nt * 8 + g < nh)
              raw[i] = *reinterpret_cast<const uint2*>(p.q + (int64_t)b * p.q_stride +
                                                       (int64_t)(kh * p.G + h0 + nt * 8 + g) * D + 16 * i + 4 * c);
          }
          const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i].x));
          const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i].y));
          amax = fmaxf(amax, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(v.x), fabsf(v.y))));
          poison = fmaf(u.x, 0.f, fmaf(u.y, 0.f, fmaf(v.x, 0.f, fmaf(v.y, 0.f, poison))));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        poison += __shfl_xor_sync(0xffffffffu, poison, 1);
        poison += __shfl_xor_sync(0xffffffffu, poison, 2);
        const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -90), 127) - (E4M3 ? 11 : 21);
        const float f = __uint_as_float((uint32_t)(127 - e) << 23);
        const float back = fmaf(__uint_as_float((uint32_t)(127 + e) << 23), p.scale_log2, poison);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i].x));
          const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i].y));
          const float x[4] = {u.x * f, u.y * f, v.x * f, v.y * f};
          if constexpr (E4M3) {
            const __half2 hu = __floats2half2_rn(x[0], x[1]), hv = __floats2half2_rn(x[2], x[3]);
            qf[nt][i][0] = *reinterpret_cast<const uint32_t*>(&hu);
            qf[nt][i][1] = *reinterpret_cast<const uint32_t*>(&hv);
          } else {
            qf[nt][i][0] = qf[nt][i][1] = qf[nt][i][2] = 0u;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int q0 = __float2int_rn(x[k]), q1 = (q0 - (int8_t)q0) >> 8, q2 = (q1 - (int8_t)q1) >> 8;
              qf[nt][i][0] |= (uint32_t)(q0 & 0xff) << (8 * k);
              qf[nt][i][1] |= (uint32_t)(q1 & 0xff) << (8 * k);
              qf[nt][i][2] |= (uint32_t)(q2 & 0xff) << (8 * k);
            }
          }
        }
        qmul[nt][0] = __shfl_sync(0xffffffffu, back, 8 * c);  // columns 2 c and 2 c + 1
        qmul[nt][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < OWN; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[i][nt][k] = 0.f;
      }
    }

    // scores of this warp's 16 tokens
    float s[TW][NT][4], vs[TW], ev[TW];
    bool up = false;
#pragma unroll
    for (int q = 0; q < TW; ++q) {
      const int tile = tok0 + (warp * TW + q) * 16, tok = tile + g;
      using Acc = typename std::conditional<E4M3, float, int>::type;
      Acc acc[NT][PL][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < PL * 4; ++e) acc[nt][e / 4][e % 4] = 0;
      const uint32_t kb = st + ((warp * TW + q) * 16 + frow) * S::kRow;
#pragma unroll
      for (int j2 = 0; j2 < CH / 2; ++j2) {
        uint32_t r[4];  // rows 0-7 and 8-15 of chunk 2 j2, then of the next one
        ldsm4(r, kb + ((S::kSwizzle ? (2 * j2) ^ (fhi ^ (frow & 7)) : 2 * j2 + fhi) << 4));
        if constexpr (E4M3) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t a[4];
            expand4<E4M3, false>(r[2 * i], a[0], a[2]);
            expand4<E4M3, false>(r[2 * i + 1], a[1], a[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(acc[nt][i], a, qf[nt][2 * j2 + i][0], qf[nt][2 * j2 + i][1]);
          }
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pl = 0; pl < PL; ++pl) mma_s8(acc[nt][pl], r, qf[nt][2 * j2][pl], qf[nt][2 * j2 + 1][pl]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if constexpr (E4M3)
            s[q][nt][e] = acc[nt][0][e] + acc[nt][1][e];
          else
            s[q][nt][e] = fmaf((float)acc[nt][PL - 1][e], 65536.f, fmaf((float)acc[nt][1][e], 256.f, (float)acc[nt][0][e]));
      float ks;
      asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(ks), "=f"(vs[q]) : "r"(tail + 8 * (warp * TW + q)) : "memory");
      if (tile >= cur.r.L) vs[q] = 0.f;  // no token here: whatever scale was read, the probabilities are 0
      ev[q] = (float)max((int)((__float_as_uint(vs[q]) >> 23) & 0xff) - 127, -100);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[q][nt][e] *= ks * qmul[nt][e & 1];
      if (p.cap > 0.f) {  // cap * tanh(x / cap) = cap * (1 - 2 / (1 + e^(2 x / cap)))
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[q][nt][e] = p.cap_log2 * (1.f - __fdividef(2.f, 1.f + ex2(s[q][nt][e] * p.cap)));
      }
      bool ok0 = true, ok1 = true;
      if (tile < cur.r.lo || tile + 16 > cur.r.L) {
        ok0 = tok >= cur.r.lo && tok < cur.r.L, ok1 = tok + 8 >= cur.r.lo && tok + 8 < cur.r.L;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[q][nt][e] = (e < 2 ? ok0 : ok1) ? s[q][nt][e] : -INFINITY;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        up |= fmaxf(s[q][nt][0], s[q][nt][2]) + ev[q] > m[nt][0] + kSlack ||
              fmaxf(s[q][nt][1], s[q][nt][3]) + ev[q] > m[nt][1] + kSlack;
      if constexpr (MASS) {
        float* sc = p.scores + ((int64_t)(b * p.Hk + kh) * (p.mb << p.bs_log2) + tok) * p.G + h0;
        const bool pairs = (p.G & 1) == 0;  // a token's scores of two heads lie at a multiple of 8 bytes
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int hh = nt * 8 + 2 * c;
            float* d = sc + (e < 2 ? 0 : 8 * p.G) + hh;
            if (!(e < 2 ? ok0 : ok1) || hh >= nh) continue;
            if (pairs) {
              *reinterpret_cast<float2*>(d) = make_float2(s[q][nt][e], s[q][nt][e + 1]);
            } else {
              d[0] = s[q][nt][e];
              if (hh + 1 < nh) d[1] = s[q][nt][e + 1];
            }
          }
      }
    }
    // probabilities in f16 (2^-11 relative): the output's bf16 rounding is eight times coarser
    const uint32_t pd = psm + g * S::kPRow + warp * TW * 32 + 4 * c;
    float sum[NT][2];
    auto put = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
        for (int q = 0; q < TW; ++q) {
          float e4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) e4[e] = ex2_twice(fmaf(s[q][nt][e], 0.5f, -0.5f * m[nt][e & 1]));  // a masked score is -inf
          sum[nt][0] += e4[0] + e4[2];
          sum[nt][1] += e4[1] + e4[3];
          const __half2 u = __floats2half2_rn(e4[0] * vs[q], e4[1] * vs[q]);
          const __half2 v = __floats2half2_rn(e4[2] * vs[q], e4[3] * vs[q]);
          const uint32_t x0 = movm_t(*reinterpret_cast<const uint32_t*>(&u));  // now tokens 2 c, 2 c + 1 of head g
          const uint32_t x1 = movm_t(*reinterpret_cast<const uint32_t*>(&v));
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(pd + nt * 8 * S::kPRow + q * 32), "r"(x0) : "memory");
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(pd + nt * 8 * S::kPRow + q * 32 + 16), "r"(x1) : "memory");
        }
      }
    };
    put();
    if (__syncthreads_or(up)) {  // a score passed the reference: take the step's true maximum
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float y = -INFINITY;
#pragma unroll
          for (int q = 0; q < TW; ++q) y = fmaxf(y, fmaxf(s[q][nt][e], s[q][nt][e + 2]) + ev[q]);
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
          y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
          if (g == 0) sm_x[warp][nt * 8 + 2 * c + e] = y;
        }
      __syncthreads();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float y = m[nt][e];
#pragma unroll
          for (int w = 0; w < W; ++w) y = fmaxf(y, sm_x[w][nt * 8 + 2 * c + e]);
          const float d = y > m[nt][e] ? m[nt][e] - y : 0.f, al = ex2(d);
          m[nt][e] = y;
          l[nt][e] = shift_sum(l[nt][e], d);
#pragma unroll
          for (int i = 0; i < OWN; ++i) o[i][nt][e] *= al, o[i][nt][e + 2] *= al;
        }
      put();
      __syncthreads();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) l[nt][0] += sum[nt][0], l[nt][1] += sum[nt][1];

    // O^T of this warp's dims over the step's tokens, two tiles at a time (tiles behind L are zero)
#pragma unroll
    for (int t2 = 0; t2 < T / 32; ++t2) {
      uint32_t pb[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) ldsm4(pb[nt], psm + (nt * 8 + (lane & 7)) * S::kPRow + t2 * 64 + (lane >> 3) * 16);
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        uint32_t r[4], a[4];
        const int row = t2 * 32 + (lane & 7) + (lane >> 3) * 8, ch = warp * OWN + i;
        ldsm4_t(r, st + S::kSide + row * S::kRow + ((S::kSwizzle ? ch ^ (row & 7) : ch) << 4));
        expand4<E4M3, true>(r[0], a[0], a[1]);
        expand4<E4M3, true>(r[1], a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(o[i][nt], a, pb[nt][0], pb[nt][1]);
        expand4<E4M3, true>(r[2], a[0], a[1]);
        expand4<E4M3, true>(r[3], a[2], a[3]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(o[i][nt], a, pb[nt][2], pb[nt][3]);
      }
    }

    st = st == ring + (S::kStages - 1) * S::kStage ? ring : st + S::kStage;
    const int step = cur.s++;
    const bool last = cur.s == cur.r.n;
    if (!last && j + 1 < count) continue;
    // the head tile ends here, or goes on in the next CTA's stretch
    const bool whole = begun && last;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float y = l[nt][e];
        y += __shfl_xor_sync(0xffffffffu, y, 4);
        y += __shfl_xor_sync(0xffffffffu, y, 8);
        y += __shfl_xor_sync(0xffffffffu, y, 16);
        if (g == 0) sm_l[warp][nt * 8 + 2 * c + e] = y;
      }
    __syncthreads();
    const uint32_t part = blockIdx.x * 2 + (j > step ? 1 : 0);  // 0: it holds the stretch's first step
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int hh = nt * 8 + 2 * c + e;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += sm_l[w][hh];
        if (hh >= nh) continue;
        const int64_t row = (int64_t)b * p.H + kh * p.G + h0 + hh;
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          const int d = (warp * OWN + i) * 16 + 2 * g;
          if (whole)
            *reinterpret_cast<uint32_t*>(p.out + row * D + d) = saturate2(pack_bf16x2(o[i][nt][e] * inv, o[i][nt][e + 2] * inv));
          else
            *reinterpret_cast<float2*>(p.part_o + ((int64_t)part * HB + hh) * D + d) = make_float2(o[i][nt][e], o[i][nt][e + 2]);
        }
        if (warp == 0 && g == 0) {
          if (!whole) *reinterpret_cast<float2*>(p.part_ml + ((int64_t)part * HB + hh) * 2) = make_float2(m[nt][e], sum);
          else if (MASS) *reinterpret_cast<float2*>(p.row_ml + row * 2) = make_float2(m[nt][e], sum);
        }
      }
    if (begun && threadIdx.x == 0) {  // the CTA that holds the first step says how many parts there are
      int parts = 1;
      if (!last) {
        parts = (int)(stretch_of(first + j - step + cur.r.n - 1, total, grid) - blockIdx.x) + 1;
        *reinterpret_cast<int4*>(p.splits + (int64_t)blockIdx.x * 4) = make_int4(b, kh * p.NG + cur.hg, (int)part, parts);
      }
      if (MASS) *reinterpret_cast<int2*>(p.spans + ((int64_t)b * X + kh * p.NG + cur.hg) * 2) = make_int2((int)part, parts);
    }
    if (last) next_head(cur, p, T);
  }
  cp_async_wait<0>();
}

// Part number i of a head tile: its first one, then the first slots of the CTAs that follow.
GOLLEK_DEVICE int64_t part_slot(int first, int i) { return i == 0 ? first : (first & ~1) + 2 * i; }

// Reference and sum of head hh over a head tile's n parts, by one warp.
GOLLEK_DEVICE float2 join_ml(const DecArgs& p, int first, int n, int HB, int hh) {
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  const int lane = threadIdx.x & 31;
  float2 x = make_float2(-INFINITY, 0.f);
  if (lane < n) x = ml[part_slot(first, lane) * HB + hh];
  float M = x.x;
  for (int i = lane + 32; i < n; i += 32) M = fmaxf(M, ml[part_slot(first, i) * HB + hh].x);
  M = warp_max(M);
  float sum = x.x == -INFINITY ? 0.f : shift_sum(x.y, x.x - M);
  for (int i = lane + 32; i < n; i += 32) {
    const float2 y = ml[part_slot(first, i) * HB + hh];
    if (y.x != -INFINITY) sum += shift_sum(y.y, y.x - M);
  }
  return make_float2(M, warp_sum(sum));
}

// Joins the parts of the head tiles that several CTAs shared: CTA c < grid the one that leaves the decode kernel's
// CTA c; the others add the softmax weights of the batch's pieces (row, kv head, kMassTokens tokens) to mass, summed over
// the head group in head order: a CTA for each of the `tiles` pieces that a full table would hold, or (0: those would be
// more than 16 an SM, several times what it holds at once) the pieces that the lengths have in turn. An entry gets one add
// per call, so sums do not depend on the order of the CTAs unless rows share a block.
// Measured: the weights of 64 rows of up to 4k, 32 heads, add 16 us to the 61 us of the attention: 20 MB of scores, 4 bytes a head
// and token, go out and come back (3 us each way at most), but this pass begins when the whole decode kernel has ended and loads
// block ids, scores and sums one behind the other. Under a table 32 times wider than the rows: 101 us by events, where a
// CTA for every piece of the table took 153 us; where the pieces fit the grid, to search for them costs 2 us (87 us, not 85).
constexpr int kJoinThreads = 256, kMassTokens = 1024;

// The weights of kMassTokens tokens from `first` on of a row and KV head, by a CTA; sm: a float for each head of the group.
template <int GV>  // heads per KV head where they are 1, 2, 4 or 8, else 0
GOLLEK_DEVICE void weigh_piece(const DecArgs& p, const DecRow& r, int b, int kh, int first, int HB, float* sm) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, X = p.Hk * p.NG;
  const float* sc = p.scores + ((int64_t)b * p.Hk + kh) * (p.mb << p.bs_log2) * p.G;
  const int* bt = p.tables + (int64_t)b * p.bt_stride;
  float* mass = p.mass + (kh << p.bs_log2);
  const int row = p.Hk << p.bs_log2, mask = (1 << p.bs_log2) - 1;
  constexpr int GN = GV > 0 ? GV : 1, N = kMassTokens / kJoinThreads;
  // the tokens' scores and blocks are on their way while the heads' sums are joined
  float v[N][GN];
  int id[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int t = first + threadIdx.x + k * kJoinThreads;
    id[k] = t >= r.lo && t < r.L ? checked_index(bt[t >> p.bs_log2], p.num_blocks, p.bounds, -1) : -1;  // beyond the pool: none
    if (GV > 0 && id[k] >= 0) {
      if constexpr (GV == 1) v[k][0] = sc[t];
      if constexpr (GV == 2) *reinterpret_cast<float2*>(v[k]) = reinterpret_cast<const float2*>(sc)[t];
      if constexpr (GV >= 4)
#pragma unroll
        for (int h = 0; h < GV; h += 4) *reinterpret_cast<float4*>(v[k] + h) = reinterpret_cast<const float4*>(sc)[((int64_t)t * GV + h) / 4];
    }
  }
  for (int h = warp; h < p.G; h += kJoinThreads / 32) {
    const int2 span = reinterpret_cast<const int2*>(p.spans)[(int64_t)b * X + kh * p.NG + h / HB];
    const float2 ml = span.y == 1 ? reinterpret_cast<const float2*>(p.row_ml)[(int64_t)b * p.H + kh * p.G + h]
                                  : join_ml(p, span.x, span.y, HB, h % HB);
    if (lane == 0) sm[h] = ml.x + log2f(ml.y);
  }
  __syncthreads();
  float lse[GN];
#pragma unroll
  for (int h = 0; h < GN; ++h) lse[h] = sm[h];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (id[k] < 0) continue;
    const int t = first + threadIdx.x + k * kJoinThreads;
    float w = 0.f;
    if constexpr (GV > 0) {
#pragma unroll
      for (int h = 0; h < GN; ++h) w += ex2(v[k][h] - lse[h]);
    } else {
      for (int h = 0; h < p.G; ++h) w += ex2(sc[(int64_t)t * p.G + h] - sm[h]);
    }
    atomicAdd(mass + (int64_t)id[k] * row + (t & mask), w);
  }
}

template <int GV>  // as weigh_piece's; -1: no weights
__global__ void __launch_bounds__(kJoinThreads) block8_join_kernel(const DecArgs p, int D, int HB, int tiles) {
  __shared__ float sm[128];
  __shared__ float4 others[kJoinThreads];
  __shared__ float2 others_ml[kJoinThreads];
  if (GV < 0 || (int)blockIdx.x < p.grid) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the decode kernel still runs
    const int4 sp = *reinterpret_cast<const int4*>(p.splits + blockIdx.x * 4);  // row, head tile, first part, parts
    if (sp.x < 0) return;
    const int kh = sp.y / p.NG, h0 = (sp.y - kh * p.NG) * HB, nh = min(p.G - h0, HB);
    // a thread takes four dims of a head; where they leave threads over, those share the parts
    const int quads = nh * D / 4, groups = max(1, kJoinThreads / quads);
    __nv_bfloat16* out = p.out + ((int64_t)sp.x * p.H + kh * p.G + h0) * D;
    for (int q0 = 0; q0 < quads; q0 += kJoinThreads) {
      const int gr = threadIdx.x / quads, q = q0 + (groups > 1 ? threadIdx.x % quads : threadIdx.x);
      float M = -INFINITY, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      auto add = [&](const float2& ml, const float4& o) {
        const float m = fmaxf(M, ml.x), d0 = m == -INFINITY ? 0.f : M - m, d1 = m == -INFINITY ? 0.f : ml.x - m;
        const float f0 = ex2(d0), f1 = ex2(d1);
        M = m;
        sum = shift_sum(sum, d0) + shift_sum(ml.y, d1);
        acc.x = f0 * acc.x + f1 * o.x;
        acc.y = f0 * acc.y + f1 * o.y;
        acc.z = f0 * acc.z + f1 * o.z;
        acc.w = f0 * acc.w + f1 * o.w;
      };
      if (q < quads && (groups == 1 || gr < groups)) {
        const int hh = q * 4 / D;
        constexpr int N = 4;  // parts whose loads are in flight together
        for (int i = groups > 1 ? gr : 0; i < sp.w; i += N * groups) {
          float2 ml[N];
          float4 o[N];
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int64_t k = part_slot(sp.z, min(i + e * groups, sp.w - 1)) * HB + hh;
            ml[e] = reinterpret_cast<const float2*>(p.part_ml)[k];
            o[e] = *reinterpret_cast<const float4*>(p.part_o + k * D + (q * 4 - hh * D));
          }
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (i + e * groups < sp.w) add(ml[e], o[e]);
        }
      }
      if (groups > 1) {
        if (gr > 0 && gr < groups) others[threadIdx.x] = acc, others_ml[threadIdx.x] = make_float2(M, sum);
        __syncthreads();
        if (gr > 0) return;
        for (int g = 1; g < groups; ++g) add(others_ml[threadIdx.x + g * quads], others[threadIdx.x + g * quads]);
      }
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
      if (q < quads)
        *reinterpret_cast<uint2*>(out + q * 4) =
            make_uint2(saturate2(pack_bf16x2(acc.x * inv, acc.y * inv)), saturate2(pack_bf16x2(acc.z * inv, acc.w * inv)));
    }
    return;
  }
  if constexpr (GV >= 0) {
    if (tiles > 0) {
      const int x = (int)blockIdx.x - p.grid, bk = x / tiles, b = bk / p.Hk, first = (x - bk * tiles) * kMassTokens;
      const DecRow r = dec_row(p, b, kMassTokens);
      if (first >= r.L || first + kMassTokens <= r.lo) return;
      asm volatile("griddepcontrol.wait;" ::: "memory");
      weigh_piece<GV>(p, r, b, bk - b * p.Hk, first, HB, sm);
      return;
    }
    auto row_pieces = [&](int b) { return dec_row(p, b, kMassTokens).n; };
    const RowList<decltype(row_pieces)> list(p.B, p.Hk, row_pieces);  // lengths are inputs: no wait
    bool waited = false;
    for (int64_t x = (int)blockIdx.x - p.grid; x < list.total; x += (int)gridDim.x - p.grid) {
      int64_t place = x;
      const int b = list.find(place);
      const DecRow r = dec_row(p, b, kMassTokens);
      if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
      else __syncthreads();  // the last piece's readers of sm are done
      waited = true;
      weigh_piece<GV>(p, r, b, (int)(place / r.n), r.t0 + (int)(place % r.n) * kMassTokens, HB, sm);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Eviction, step 1: which tokens stay. One CTA per (layer, sequence, kv head).
//
// Of a sequence with L tokens and K < L to keep: the first a = min(sink, K), the last
// r = min(recent, K - a), and of those between the K - a - r with the largest mass (ties: the lower
// index). A radix select (11 + 11 + 10 bits of the order-preserving integer of the mass) finds the
// smallest mass that stays and how many tokens of exactly that mass do; one ordered pass lists them.
// Measured: 192 (layer, sequence, head) of 8192 tokens 20 us, bound by the latency of the four passes over a row.
// ---------------------------------------------------------------------------------------------
constexpr int kSelThreads = 512;
constexpr int kSelKeys = 16384;  // masses held in shared memory; longer sequences read them again per pass

struct EvictArgs {
  uint8_t* cache;
  float* scales;
  float* mass;
  const int* tables;
  const int* lens;
  const int* keep;
  int* kept;  // [layers, B, Hk, max_keep]
  int64_t bt_stride;
  int layers, B, Hk, D, mb, bs_log2, num_blocks, sink, recent, max_keep;
  uint32_t* bounds;
};

struct EvictRow {
  int L, K;
  bool cut;
};
GOLLEK_DEVICE EvictRow evict_row(const EvictArgs& p, int b) {
  EvictRow r;
  r.L = min(max(p.lens[b], 0), p.mb << p.bs_log2);
  r.K = min(max(p.keep[b], 0), r.L);
  r.cut = r.K < r.L;
  if (r.cut) r.K = min(r.K, p.max_keep);
  return r;
}

GOLLEK_DEVICE uint32_t mass_key(float f) {  // NaN counts as 0, -0 as 0, infinities as the largest number
  f = f == f ? fminf(fmaxf(f, -3.402823466e38f), 3.402823466e38f) + 0.f : 0.f;
  const uint32_t u = __float_as_uint(f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// exclusive prefix sum of one value per thread; `total` is the sum
GOLLEK_DEVICE uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const uint32_t y = warp_sums[w];
    if (w < warp) before += y;
    total += y;
  }
  return before + x - v;
}

__global__ void __launch_bounds__(kSelThreads) kv_evict_select_kernel(const EvictArgs p) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t hist[2048], warp_sums[kSelThreads / 32], found[2];
  __shared__ uint2 counts[kSelThreads / 32];
  asm volatile("griddepcontrol.launch_dependents;");
  const int h = blockIdx.x, b = blockIdx.y, ly = blockIdx.z;
  const EvictRow r = evict_row(p, b);
  int* kept = p.kept + (((int64_t)ly * p.B + b) * p.Hk + h) * p.max_keep;
  if (!r.cut) {
    for (int i = threadIdx.x; i < p.max_keep; i += kSelThreads) kept[i] = i < r.L ? i : -1;
    return;
  }
  const int a = min(p.sink, r.K), rec = min(p.recent, r.K - a);
  const int c0 = a, n = r.L - rec - a, take = r.K - a - rec;  // candidates [c0, c0 + n)
  for (int i = threadIdx.x; i < p.max_keep; i += kSelThreads)
    if (i < a) kept[i] = i;
    else if (i >= r.K) kept[i] = -1;
    else if (i >= r.K - rec) kept[i] = r.L - r.K + i;
  if (take <= 0) return;
  const float* mass = p.mass + (int64_t)ly * p.num_blocks * p.Hk * (1 << p.bs_log2);
  const int* bt = p.tables + (int64_t)b * p.bt_stride;
  auto load = [&](int i) {
    const int t = c0 + i;
    const int64_t id = checked_index(bt[t >> p.bs_log2], p.num_blocks, p.bounds);
    return mass_key(mass[((id * p.Hk + h) << p.bs_log2) + (t & ((1 << p.bs_log2) - 1))]);
  };
  const bool held = n <= kSelKeys;
  if (held)
    for (int i = threadIdx.x; i < n; i += kSelThreads) keys[i] = load(i);
  uint32_t prefix = 0;   // the bits of the threshold found so far
  uint32_t want = take;  // rank still sought among the keys that share them
  int bits_done = 0;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int width = pass < 2 ? 11 : 10, shift = 32 - bits_done - width;
    for (int i = threadIdx.x; i < 2048; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kSelThreads) {
      const uint32_t k = held ? keys[i] : load(i);
      if (bits_done == 0 || (k >> (32 - bits_done)) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << width) - 1)], 1u);
    }
    __syncthreads();
    // four bins a thread, from the top: the bin where the count from above reaches `want`
    const int bin0 = 2047 - 4 * threadIdx.x;
    const uint32_t h0 = hist[bin0], h1 = hist[bin0 - 1], h2 = hist[bin0 - 2], h3 = hist[bin0 - 3];
    uint32_t total;
    uint32_t above = block_scan(h0 + h1 + h2 + h3, warp_sums, total);
    const uint32_t hb[4] = {h0, h1, h2, h3};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (above < want && above + hb[k] >= want) found[0] = bin0 - k, found[1] = want - above;
      above += hb[k];
    }
    __syncthreads();
    prefix = (prefix << width) | found[0];
    want = found[1];
    bits_done += width;
    __syncthreads();
  }
  // prefix is the smallest key that stays, `want` how many tokens with it do (the first ones). Every warp counts
  // a stretch of the candidates, then lists it behind the stretches before.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kSelThreads / 32;
  const int per = ((n + warps - 1) / warps + 31) & ~31, i0 = min(n, warp * per), i1 = min(n, i0 + per);
  uint32_t gt = 0, eq = 0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const uint32_t k = i < i1 ? (held ? keys[i] : load(i)) : 0u;
    gt += __popc(__ballot_sync(0xffffffffu, i < i1 && k > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, i < i1 && k == prefix));
  }
  if (lane == 0) counts[warp] = make_uint2(gt, eq);
  __syncthreads();
  gt = eq = 0;
  for (int w = 0; w < warp; ++w) gt += counts[w].x, eq += counts[w].y;
  const uint32_t before = (1u << lane) - 1;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const uint32_t k = i < i1 ? (held ? keys[i] : load(i)) : 0u;
    const uint32_t bg = __ballot_sync(0xffffffffu, i < i1 && k > prefix), be = __ballot_sync(0xffffffffu, i < i1 && k == prefix);
    const uint32_t g = gt + __popc(bg & before), e = eq + __popc(be & before);
    if (((bg >> lane) & 1) || (((be >> lane) & 1) && e < want)) kept[a + g + min(e, want)] = c0 + i;
    gt += __popc(bg);
    eq += __popc(be);
  }
}

// ---------------------------------------------------------------------------------------------
// Eviction, step 2: the kept tokens move to the front, in order. One CTA per (layer, sequence, kv head, K / V / mass).
//
// In place: kept[j] >= j, so a chunk's sources lie at or behind its own places. A chunk may be read as early as one likes
// (what goes before it is written in front of it), and must be read before it or any later one is written: chunks go
// up, and a chunk's loads end before a barrier that its stores follow. So codes are read two chunks ahead (cp.async
// into a ring; a thread only touches the codes that it loaded itself), the indices and block ids they hang on earlier
// still. Each destination block gets the smallest power-of-two scale for what it then holds: one barrier a chunk, for its
// largest magnitude.
// Measured: 8 layers x 4 sequences of 8192 tokens to 60 % (8 heads of 128, e4m3; 660 MB at least) 176 us with step 1 where
// earlier evictions have drawn the rows' survivors together, 202 us for the first one of rows as they were written. A (layer,
// sequence, head) is one chain of chunks, and 512 chains are three or four an SM: latency. With two threads a token, whose
// loads and stores touch 32 bytes of 16 rows at a time, the way to L2 was the bound (209 us); copies by the bulk engine, a row
// each, took 313 us.
// ---------------------------------------------------------------------------------------------
// A magnitude costs one instruction a value (packed 16-bit maxima), a change of scale by a power of two two, all exact.
constexpr int kMoveThreads = 256;
constexpr int kMoveStages = 3;

// Running maximum magnitude of four codes each in two 16-bit lanes: hi and lo of int8, magnitude bits of e4m3.
template <bool E4M3>
struct Top4 {
  uint32_t hi = 0, lo = 0;
  GOLLEK_DEVICE void add(uint32_t w) {
    if constexpr (E4M3) {  // the bits below the sign order like the magnitudes
      hi = __vimax3_u16x2(hi, w & 0x007f007fu, (w >> 8) & 0x007f007fu);
    } else {  // bytes sign-extended to 16 bits
      uint32_t e, o;
      asm("prmt.b32 %0, %1, 0, 0xa280;" : "=r"(e) : "r"(w));
      asm("prmt.b32 %0, %1, 0, 0xb391;" : "=r"(o) : "r"(w));
      hi = __vimax3_s16x2(hi, e, o);
      lo = __vimin3_s16x2(lo, e, o);
    }
  }
  GOLLEK_DEVICE float value() const {
    if constexpr (E4M3) {
      float f[4];
      decode4<true>(max(hi & 0xffffu, hi >> 16), f);
      return f[0];
    } else {
      const int a = max((int)(int16_t)hi, (int)(int16_t)(hi >> 16)), b = min((int)(int16_t)lo, (int)(int16_t)(lo >> 16));
      return (float)max(a, -b);
    }
  }
};

// Codes times a ratio of scales. A power of two within f16's reach goes through f16 exactly: e4m3 by a product, int8 by
// one fma on 1152 + code whose sum with 1536 rounds to the integer (ties to even); others go through fp32.
template <bool E4M3, int N>
GOLLEK_DEVICE void rescale(uint32_t* w, float ratio) {
  if (ratio == 1.f) return;
  const uint32_t b = __float_as_uint(ratio);
  const int e = (int)(b >> 23) - 127;
  const __half2 m = __float2half2_rn(ratio);
  if ((b & 0x7fffffu) == 0 && (E4M3 ? e >= -14 && e <= 6 : e >= -7 && e <= 5)) {
    const __half2 c = __float2half2_rn(1536.f - 1152.f * ratio);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (E4M3) {
        uint32_t lo, hi;
        expand4<true, false>(w[i], lo, hi);
        const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&lo), m), y = __hmul2(*reinterpret_cast<const __half2*>(&hi), m);
        const uint32_t p = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&x), __NV_SATFINITE, __NV_E4M3);
        const uint32_t q = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&y), __NV_SATFINITE, __NV_E4M3);
        w[i] = p | (q << 16);
      } else {
        const uint32_t ev = (w[i] & 0x00ff00ffu) ^ 0x64806480u, od = ((w[i] >> 8) & 0x00ff00ffu) ^ 0x64806480u;
        const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&ev), m, c), y = __hfma2(*reinterpret_cast<const __half2*>(&od), m, c);
        w[i] = __byte_perm(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y), 0x6240);
      }
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      float f[4];
      decode4<E4M3>(w[i], f);
      w[i] = encode4<E4M3>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
    }
  }
}

// The masses of the kept tokens, the same way: a chunk's loads end before its stores.
GOLLEK_DEVICE void move_masses(const EvictArgs& p, const EvictRow& r, int h, int b, int ly) {
  constexpr int N = 8;
  const int* kept = p.kept + (((int64_t)ly * p.B + b) * p.Hk + h) * p.max_keep;
  const int* bt = p.tables + (int64_t)b * p.bt_stride;
  float* mass = p.mass + (((int64_t)ly * p.num_blocks * p.Hk + h) << p.bs_log2);
  const int mask = (1 << p.bs_log2) - 1;
  auto at = [&](int t, int id) { return mass + (uint64_t)(uint32_t)id * (p.Hk << p.bs_log2) + (t & mask); };
  auto from = [&](int t) { return at(t, checked_index(bt[t >> p.bs_log2], p.num_blocks, p.bounds)); };
  for (int base = threadIdx.x; base - (int)threadIdx.x < r.K; base += N * kMoveThreads) {
    float v[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (base + k * kMoveThreads < r.K) v[k] = *from(kept[base + k * kMoveThreads]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int t = base + k * kMoveThreads;
      if (t >= r.K) continue;
      const int id = checked_index(bt[t >> p.bs_log2], p.num_blocks, p.bounds, -1);
      if (id >= 0) *at(t, id) = v[k];
    }
  }
}

// A warp moves TW tokens of a chunk. Piece i of its lanes covers whole rows of R tokens, so memory sees full lines; the lanes
// keep one token's index and block id each and hand them round.
template <int D>
struct MoveShape {
  static constexpr int P = D / 16;                       // 16-byte pieces of a token
  static constexpr int R = 32 / P;                       // tokens a warp takes at once
  static constexpr int TW = D <= 64 ? 32 : D <= 128 ? 16 : 8;
  static constexpr int I = (TW + R - 1) / R;
  static constexpr int kChunk = kMoveThreads / 32 * TW;  // tokens, a multiple of every block size
  static constexpr int kStage = kMoveThreads * I * 16 + kChunk * 4;  // codes, then their scales
  static constexpr int kSmem = kMoveStages * kStage;
};

template <bool E4M3, int D>
__global__ void __launch_bounds__(kMoveThreads, 4) kv_evict_move_kernel(const EvictArgs p) {
  using S = MoveShape<D>;
  constexpr int P = S::P, R = S::R, TW = S::TW, I = S::I, kChunk = S::kChunk;
  constexpr int GR = TW > 16 ? 2 : 1;  // 16 tokens at an aligned place share a block: groups of pieces with one scale
  extern __shared__ __align__(16) uint8_t ring[];
  // largest magnitude of each destination block of a chunk (float bits): one being filled, one read, one cleared
  __shared__ uint32_t top[3][kChunk / 16];
  // masses come last: the CTAs that move codes spread over the SMs evenly
  const int h = blockIdx.x, b = blockIdx.y, ly = blockIdx.z % p.layers, w = blockIdx.z / p.layers;  // w: K, V, masses
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the choice is still being made
  const EvictRow r = evict_row(p, b);
  if (!r.cut || r.K == 0) return;
  if (w == 2) {
    move_masses(p, r, h, b, ly);
    return;
  }
  const int bs = 1 << p.bs_log2, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (r.K + kChunk - 1) / kChunk;
  const int* kept = p.kept + (((int64_t)ly * p.B + b) * p.Hk + h) * p.max_keep;
  const int* bt = p.tables + (int64_t)b * p.bt_stride;
  // a block's K (or V) of this head and its scale: base + block id * stride
  const uint32_t row_stride = (uint32_t)(2 * p.Hk << p.bs_log2) * D;
  uint8_t* codes = p.cache + ((int64_t)ly * p.num_blocks * 2 * p.Hk + w * p.Hk + h) * ((int64_t)D << p.bs_log2);
  float* scales = p.scales + (int64_t)ly * p.num_blocks * 2 * p.Hk + w * p.Hk + h;
  // beyond the pool: block 0 to read from, none to write to
  auto block_of = [&](int t, int safe) { return checked_index(bt[t >> p.bs_log2], p.num_blocks, p.bounds, safe); };
  auto scale_at = [&](int id) { return scales + (uint64_t)(uint32_t)id * (2 * p.Hk); };
  const int own = warp * TW + (lane & (TW - 1));  // the token of a chunk whose index and block ids this lane keeps
  const int piece = lane % P * 16;
  auto tok = [&](int i) { return i * R + lane / P; };  // token of the warp's that piece i belongs to
  auto mine = [&](int i) { return lane < R * P && tok(i) < TW; };

  // indices of a chunk, block ids of a chunk, codes and scales of a chunk: each one step behind the one before
  int src2, src1, id1;
  auto load_src = [&](int c) { return own < r.K - c * kChunk ? kept[c * kChunk + own] : -1; };
  auto load_id = [&](int src) { return src >= 0 ? block_of(src, 0) : 0; };
  auto load_codes = [&](int c, int src, int id) {
    const uint32_t st = smem_u32(ring) + (c % kMoveStages) * S::kStage;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int t = __shfl_sync(0xffffffffu, src, tok(i) & 31), d = __shfl_sync(0xffffffffu, id, tok(i) & 31);
      if (mine(i) && t >= 0)
        cp_async16<0, 0>(st + (i * kMoveThreads + threadIdx.x) * 16,
                         codes + (uint64_t)(uint32_t)d * row_stride + (t & (bs - 1)) * D + piece);
    }
    if (src >= 0 && lane < TW) cp_async4(st + kMoveThreads * I * 16 + own * 4, scale_at(id));
    cp_async_commit();
  };
  if (threadIdx.x < kChunk / 16) top[0][threadIdx.x] = 0u;
  // chunk 0 and 1's codes on their way, chunk 2's ids and chunk 3's indices too
  src2 = load_src(0);
  src1 = load_src(1);
  id1 = load_id(src2);
  load_codes(0, src2, id1);
  id1 = load_id(src1);
  load_codes(1, src1, id1);
  src1 = load_src(2);
  src2 = load_src(3);
  id1 = load_id(src1);
  __syncthreads();
  for (int c = 0; c < chunks; ++c) {
    const int base = c * kChunk, n = min(kChunk, r.K - base);
    load_codes(c + 2, src1, id1);
    const int to_id = own < n ? block_of(base + own, -1) : -1;  // destination block
    src1 = src2;
    id1 = load_id(src1);
    src2 = load_src(c + 4);
    cp_async_wait<2>();
    __syncwarp();  // a token's scale is another lane's copy
    uint32_t code[I][4];
    float sc[I];
    const uint8_t* st = ring + (c % kMoveStages) * S::kStage;
    uint32_t* tp = top[c % 3];
    uint32_t amax[GR];
#pragma unroll
    for (int q = 0; q < GR; ++q) amax[q] = 0u;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if (!mine(i) || warp * TW + tok(i) >= n) continue;
      Top4<E4M3> t;
      const uint4 x = reinterpret_cast<const uint4*>(st)[i * kMoveThreads + threadIdx.x];
      code[i][0] = x.x, code[i][1] = x.y, code[i][2] = x.z, code[i][3] = x.w;
#pragma unroll
      for (int k = 0; k < 4; ++k) t.add(code[i][k]);
      sc[i] = reinterpret_cast<const float*>(st + kMoveThreads * I * 16)[warp * TW + tok(i)];
      amax[i * R / 16 % GR] = max(amax[i * R / 16 % GR], __float_as_uint(t.value() * sc[i]));
    }
#pragma unroll
    for (int q = 0; q < GR; ++q) {
      amax[q] = __reduce_max_sync(0xffffffffu, amax[q]);
      if (lane == 0) atomicMax(&tp[(warp * TW + 16 * q) >> p.bs_log2], amax[q]);
    }
    if (threadIdx.x < kChunk / 16) top[(c + 1) % 3][threadIdx.x] = 0u;  // its readers are behind the last barrier, its writers the next
    __syncthreads();
    float s[GR];
#pragma unroll
    for (int q = 0; q < GR; ++q) s[q] = pow2_scale<E4M3>(__uint_as_float(tp[(warp * TW + 16 * q) >> p.bs_log2]));
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int d = __shfl_sync(0xffffffffu, to_id, tok(i) & 31), to = base + warp * TW + tok(i);
      if (!mine(i) || to - base >= n || d < 0) continue;
      const float z = s[i * R / 16 % GR];
      // sc / z, z = 2^e. A code that is not zero has a ratio of 2^18 at most; beside a scale of 2^120, zeros would meet an infinity
      rescale<E4M3, 4>(code[i], fminf(sc[i] * __uint_as_float((254u << 23) - __float_as_uint(z)), 0x1p100f));
      *reinterpret_cast<uint4*>(codes + (uint64_t)(uint32_t)d * row_stride + (to & (bs - 1)) * D + piece) =
          make_uint4(code[i][0], code[i][1], code[i][2], code[i][3]);
      if ((to & (bs - 1)) == 0 && piece == 0) *scale_at(d) = z;
    }
  }
  cp_async_wait<0>();
}

// Raises a kernel's shared-memory limit once per device (the attribute lasts as long as the context).
template <auto Kernel>
void max_smem_once(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  GOLLEK_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 64 && ((done.load(std::memory_order_relaxed) >> dev) & 1)) return;
  GOLLEK_CUDA_CHECK(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
}

int log2_block(int bs) {
  throw_if(bs != 16 && bs != 32 && bs != 64, "block-scaled KV cache: block size 16, 32 or 64");
  return bs == 16 ? 4 : bs == 32 ? 5 : 6;
}

}  // namespace

void launch_kv_quant_blocks(const void* kv, int64_t st, int64_t sw, int64_t sh, const int* slots, void* cache,
                            float* scales, float* mass, int T, int Hk, int D, int bs, int num_blocks, bool e4m3,
                            cudaStream_t s) {
  QuantArgs p{reinterpret_cast<const __nv_bfloat16*>(kv), st, sw, sh, slots, reinterpret_cast<uint8_t*>(cache), scales, mass,
              T, Hk, log2_block(bs), num_blocks, 1, bounds_status()};
  if (T == 0) return;
  p.g = T >= 1024 ? 16 : 1;  // about one run of a prompt, one row of a decode step
  const int64_t warps = (int64_t)((T + p.g - 1) / p.g) * 2 * Hk;
  const unsigned grid = (unsigned)((warps + kQuantThreads / 32 - 1) / (kQuantThreads / 32));
#define GOLLEK_QB(DD)                                                        \
  if (D == DD) {                                                             \
    if (e4m3) kv_quant_blocks_kernel<true, DD><<<grid, kQuantThreads, 0, s>>>(p);\
    else kv_quant_blocks_kernel<false, DD><<<grid, kQuantThreads, 0, s>>>(p);\
    check_launch("kv_quant_blocks");                                         \
    return;                                                                  \
  }
  GOLLEK_QB(32)
  GOLLEK_QB(64)
  GOLLEK_QB(96)
  GOLLEK_QB(128)
  GOLLEK_QB(256)
#undef GOLLEK_QB
  throw_if(true, "block-scaled KV cache: unsupported head_dim " + std::to_string(D));
}

void launch_kv_dequant_scaled(const void* cache, const float* scales, const int* tables, int64_t bt_stride,
                              const int* lens, int rows, int mb, int num_blocks, int Hk, int D, int bs, bool e4m3,
                              void* dst, cudaStream_t s, const PromptRows& prompt) {
  const int lb = log2_block(bs);
  throw_if(rows > 65535, "kv_dequant_blocks: at most 65535 sequences");
  if (rows == 0 || mb == 0) return;
  auto of = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    return e4m3 ? kv_dequant_scaled_kernel<true, DD> : kv_dequant_scaled_kernel<false, DD>;
  };
  throw_if(D != 32 && D != 64 && D != 96 && D != 128 && D != 256, "block-scaled KV cache: unsupported head_dim " + std::to_string(D));
  auto k = D == 32    ? of(std::integral_constant<int, 32>{})
           : D == 64  ? of(std::integral_constant<int, 64>{})
           : D == 96  ? of(std::integral_constant<int, 96>{})
           : D == 128 ? of(std::integral_constant<int, 128>{})
                      : of(std::integral_constant<int, 256>{});
  const int mb16 = prompt.together ? (mb * bs + 127) / 128 * 8 : mb << (lb - 4);
  auto go = [&](auto... a) {  // a plan goes in front of the `together` form, whose CTAs start as it does
    if (prompt.together) launch_after(k, dim3(mb16, rows), 256, 0, s, a...);
    else k<<<dim3(mb16, rows), 256, 0, s>>>(a...);
  };
  go(reinterpret_cast<const uint8_t*>(cache), scales, tables, bt_stride, lens, mb16, mb * bs, num_blocks, Hk, lb,
     reinterpret_cast<__nv_bfloat16*>(dst), prompt, bounds_status());
  check_launch("kv_dequant_blocks");
}

namespace {

template <int D, int NT>
Block8Plan plan_for(int B, int H, int Hk, int64_t width, int splits, bool mass) {
  using S = DecShape<D, NT>;
  Block8Plan p;
  p.nt = NT;
  const int G = H / Hk, HB = 8 * NT;
  p.ng = (G + HB - 1) / HB;
  const int64_t tiles = (int64_t)B * Hk * p.ng;
  const int64_t most = tiles * ((width + S::kTokens - 1) / S::kTokens);  // steps, if every row filled its table
  const int64_t want = splits > 0 ? tiles * splits : (int64_t)device_num_sms() * S::kCtas;
  p.grid = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, most), 1 << 24));
  p.n_o = (int64_t)p.grid * 2 * HB * D;
  p.n_ml = (int64_t)p.grid * 2 * HB * 2;
  p.n_row = mass ? (int64_t)B * H * 2 : 0;
  p.n_span = (int64_t)p.grid * 4 + (mass ? tiles * 2 : 0);
  p.n_scores = mass ? (int64_t)B * H * width : 0;  // a multiple of 16, like n_o and n_ml
  return p;
}

}  // namespace

// A grid of as many CTAs as the GPU holds at once, or `splits` per (sequence, head tile) on average; never more
// than there can be steps.
Block8Plan block8_plan(int B, int H, int Hk, int D, int64_t width, int splits, bool mass) {
  throw_if(Hk <= 0 || H % Hk != 0, "block-scaled decode attention: H must be a multiple of Hk");
  throw_if(H / Hk > 128, "block-scaled decode attention: at most 128 query heads per KV head");
  const bool two = H / Hk > 8;
#define GOLLEK_B8(DD) \
  if (D == DD) return two ? plan_for<DD, 2>(B, H, Hk, width, splits, mass) : plan_for<DD, 1>(B, H, Hk, width, splits, mass);
  GOLLEK_B8(32)
  GOLLEK_B8(64)
  GOLLEK_B8(96)
  GOLLEK_B8(128)
  GOLLEK_B8(256)
#undef GOLLEK_B8
  throw std::runtime_error("block-scaled decode attention: unsupported head_dim " + std::to_string(D));
}

void launch_block8_decode(void* out, const void* q, int64_t q_stride, const void* cache, const float* scales,
                          const int* tables, int64_t bt_stride, int mb, const int* lens, int B, int H, int Hk, int D,
                          int bs, int num_blocks, const Block8Plan& plan, float scale, int window, float softcap,
                          float* workspace, float* mass, bool e4m3, cudaStream_t s) {
  DecArgs p;
  p.bs_log2 = log2_block(bs);
  if (B == 0) return;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.cache = reinterpret_cast<const uint8_t*>(cache);
  p.scales = scales;
  p.tables = tables;
  p.lens = lens;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.part_o = workspace;
  p.part_ml = p.part_o + plan.n_o;
  p.scores = p.part_ml + plan.n_ml + (int64_t)plan.grid * 4;  // behind the splits: every section a multiple of 16 bytes
  p.row_ml = p.scores + plan.n_scores;
  p.splits = reinterpret_cast<int*>(p.part_ml + plan.n_ml);
  p.spans = reinterpret_cast<int*>(p.row_ml + plan.n_row);
  p.mass = mass;
  p.q_stride = q_stride;
  p.bt_stride = bt_stride;
  p.B = B, p.H = H, p.Hk = Hk, p.G = H / Hk, p.NG = plan.ng, p.grid = plan.grid, p.mb = mb, p.num_blocks = num_blocks;
  p.window = window;
  p.scale_log2 = scale * kLog2e;
  p.cap = softcap > 0.f ? 2.f / softcap : 0.f;  // scores are in log2 units: e^(2 x / cap) = 2^(2 x log2(e) / cap)
  p.cap_log2 = softcap * kLog2e;
  p.bounds = bounds_status();
  const int64_t tiles = mass ? (((int64_t)mb << p.bs_log2) + kMassTokens - 1) / kMassTokens : 0;
  const int64_t pieces = B * Hk * tiles, most = 16 * device_num_sms();
  const int64_t join = plan.grid + std::min(pieces, most);
#define GOLLEK_B8_M(DD, NN, E, M)                                                                          \
  do {                                                                                                     \
    using S = DecShape<DD, NN>;                                                                            \
    max_smem_once<block8_decode_kernel<DD, NN, E, M>>(S::kSmem);                                           \
    block8_decode_kernel<DD, NN, E, M><<<(unsigned)plan.grid, S::kThreads, S::kSmem, s>>>(p);              \
  } while (0)
#define GOLLEK_B8_N(DD, NN)                             \
  if (e4m3) {                                           \
    if (mass) GOLLEK_B8_M(DD, NN, true, true);          \
    else GOLLEK_B8_M(DD, NN, true, false);              \
  } else {                                              \
    if (mass) GOLLEK_B8_M(DD, NN, false, true);         \
    else GOLLEK_B8_M(DD, NN, false, false);             \
  }
#define GOLLEK_B8(DD) \
  if (D == DD) {      \
    if (plan.nt == 1) { GOLLEK_B8_N(DD, 1) } else { GOLLEK_B8_N(DD, 2) } \
  }
  GOLLEK_B8(32)
  GOLLEK_B8(64)
  GOLLEK_B8(96)
  GOLLEK_B8(128)
  GOLLEK_B8(256)
#undef GOLLEK_B8
#undef GOLLEK_B8_N
#undef GOLLEK_B8_M
  check_launch("block8_decode");
  auto join_kernel = mass ? block8_join_kernel<0> : block8_join_kernel<-1>;
  if (mass && p.G == 1) join_kernel = block8_join_kernel<1>;
  if (mass && p.G == 2) join_kernel = block8_join_kernel<2>;
  if (mass && p.G == 4) join_kernel = block8_join_kernel<4>;
  if (mass && p.G == 8) join_kernel = block8_join_kernel<8>;
  launch_after(join_kernel, dim3((unsigned)join), kJoinThreads, 0, s, p, D, 8 * plan.nt,
               pieces <= most ? (int)tiles : 0);
}

void launch_kv_evict(void* cache, float* scales, float* mass, const int* tables, int64_t bt_stride, int mb,
                     const int* lens, const int* keep, int* kept, int layers, int B, int Hk, int D, int bs,
                     int num_blocks, int sink, int recent, int max_keep, bool e4m3, cudaStream_t s) {
  throw_if(D % 32 != 0 || D < 32 || D > 256, "kv_evict: head_dim must be a multiple of 32, <= 256");
  throw_if(B > 65535 || layers > 65535 / 3, "kv_evict: at most 65535 sequences and 21845 layers");
  EvictArgs p;
  p.bs_log2 = log2_block(bs);
  if (layers == 0 || B == 0 || Hk == 0) return;
  p.cache = reinterpret_cast<uint8_t*>(cache);
  p.scales = scales;
  p.mass = mass;
  p.tables = tables;
  p.lens = lens;
  p.keep = keep;
  p.kept = kept;
  p.bt_stride = bt_stride;
  p.layers = layers, p.B = B, p.Hk = Hk, p.D = D, p.mb = mb, p.num_blocks = num_blocks;
  p.sink = sink, p.recent = recent, p.max_keep = max_keep;
  p.bounds = bounds_status();
  const int smem = (int)std::min<int64_t>((int64_t)mb << p.bs_log2, kSelKeys) * 4;
  max_smem_once<kv_evict_select_kernel>(kSelKeys * 4);
  kv_evict_select_kernel<<<dim3(Hk, B, layers), kSelThreads, smem, s>>>(p);
  check_launch("kv_evict_select");
  if (max_keep == 0) return;
  auto move = [&](auto e, auto d) {
    constexpr auto k = kv_evict_move_kernel<decltype(e)::value, decltype(d)::value>;
    constexpr int smem = MoveShape<decltype(d)::value>::kSmem;
    max_smem_once<k>(smem);
    launch_after(k, dim3(Hk, B, 3 * layers), kMoveThreads, smem, s, p);
  };
  auto kind = [&](auto d) { e4m3 ? move(std::true_type{}, d) : move(std::false_type{}, d); };
  switch (D) {
    case 32: kind(std::integral_constant<int, 32>{}); break;
    case 64: kind(std::integral_constant<int, 64>{}); break;
    case 96: kind(std::integral_constant<int, 96>{}); break;
    case 128: kind(std::integral_constant<int, 128>{}); break;
    case 160: kind(std::integral_constant<int, 160>{}); break;
    case 192: kind(std::integral_constant<int, 192>{}); break;
    case 224: kind(std::integral_constant<int, 224>{}); break;
    default: kind(std::integral_constant<int, 256>{});
  }
}

}  // namespace gollek
