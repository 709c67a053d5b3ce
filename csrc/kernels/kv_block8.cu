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
// scale grows is a shift, and the bf16 copy that prompt attention reads holds every value exactly.
#include <cuda_fp8.h>

#include <algorithm>

#include "../common/common.cuh"
#include "../common/tma_host.h"
#include "launchers.h"

namespace gollek {

namespace {

constexpr float kBf16Max = 3.3895313892515355e38f;
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
// there to a raised scale, and stores the run's codes. Memory-bound: 3 bytes a value.
// ---------------------------------------------------------------------------------------------
GOLLEK_DEVICE float clean(float x) {  // NaN -> 0, infinities -> the largest bf16
  return x == x ? fminf(fmaxf(x, -kBf16Max), kBf16Max) : 0.f;
}

template <bool E4M3, int NCH>  // NCH: 4-value pieces per lane (D <= 128 * NCH)
__global__ void __launch_bounds__(256)
    kv_quant_blocks_kernel(const __nv_bfloat16* __restrict__ kv, int64_t st, int64_t sw, int64_t sh,
                           const int* __restrict__ slots, uint8_t* __restrict__ cache, float* __restrict__ scales,
                           float* __restrict__ mass, int T, int Hk, int D, int bs_log2, int num_blocks, int g,
                           uint32_t* bounds) {
  const int64_t gw = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int pair = (int)(gw % (2 * Hk));
  const int64_t grp = gw / (2 * Hk);
  const int t0 = (int)(grp * g);
  if (t0 >= T) return;
  const int w = pair / Hk, h = pair % Hk;
  const int bs = 1 << bs_log2;
  const int pieces = D >> 2;
  // lane i: slot of token t0 - 1 + i; lanes 1 .. g are this warp's tokens
  const int tl = t0 - 1 + lane;
  const int sl = (tl >= 0 && tl < T && lane <= g) ? slots[tl] : -1;
  const int bl = sl >= 0 ? sl >> bs_log2 : -1;
  const int bp = __shfl_up_sync(0xffffffffu, bl, 1);
  uint32_t leaders = __ballot_sync(0xffffffffu, lane >= 1 && bl >= 0 && bl != bp);
  while (leaders) {
    const int li = __ffs(leaders) - 1;
    leaders &= leaders - 1;
    const int tlead = t0 - 1 + li;
    const int blk = __shfl_sync(0xffffffffu, bl, li);
    // a skipped token before it: look further back for the nearest token with a slot
    int back = tlead - 1;
    while (back >= 0 && slots[back] < 0) --back;
    if (back >= 0 && (slots[back] >> bs_log2) == blk) continue;
    if (checked_index(blk, num_blocks, bounds, -1) < 0) continue;  // beyond the pool: skipped
    // pass 1: largest magnitude, offsets written
    float amax = 0.f;
    uint64_t written = 0;
    int tend = tlead;
    for (bool more = true; more && tend < T;) {
      const int s = tend + lane < T ? slots[tend + lane] : -1;
      const bool other = s >= 0 && (s >> bs_log2) != blk;
      const uint32_t om = __ballot_sync(0xffffffffu, other);
      const int n = min(T - tend, om ? __ffs(om) - 1 : 32);
      more = om == 0;
      const uint32_t valid = __ballot_sync(0xffffffffu, s >= 0 && lane < n);
      for (int i0 = 0; i0 < n; i0 += 8) {
        uint2 raw[8][NCH];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            raw[i][c] = make_uint2(0u, 0u);
            if (i0 + i < n && ((valid >> (i0 + i)) & 1) && lane + 32 * c < pieces)
              raw[i][c] = reinterpret_cast<const uint2*>(kv + (int64_t)(tend + i0 + i) * st + w * sw + h * sh)[lane + 32 * c];
          }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i][c].x));
            const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[i][c].y));
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(clean(a.x)), fabsf(clean(a.y))), fmaxf(fabsf(clean(b.x)), fabsf(clean(b.y)))));
          }
      }
      uint32_t lo = 0, hi = 0;
      if ((valid >> lane) & 1) {
        const int off = s & (bs - 1);
        if (off < 32) lo = 1u << off; else hi = 1u << (off - 32);
      }
      written |= (uint64_t)__reduce_or_sync(0xffffffffu, lo) | ((uint64_t)__reduce_or_sync(0xffffffffu, hi) << 32);
      tend += n;
    }
    amax = warp_max(amax);
    const int64_t row = ((int64_t)blk * 2 + w) * Hk + h;
    const float old = scales[row];
    const float need = pow2_scale<E4M3>(amax);
    const bool fresh = written & 1;
    const float s = fresh ? need : fmaxf(old, need);
    uint32_t* codes = reinterpret_cast<uint32_t*>(cache + (row << bs_log2) * D);
    if (!fresh && s > old) {  // the block's scale grows: round what it holds to the new one
      const float ratio = old / s;
      for (int off = 0; off < bs; ++off) {
        if ((written >> off) & 1) continue;
        for (int c = lane; c < pieces; c += 32) {
          float f[4];
          decode4<E4M3>(codes[off * pieces + c], f);
          codes[off * pieces + c] = encode4<E4M3>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
        }
      }
    }
    __syncwarp();
    if (lane == 0) scales[row] = s;
    const float inv = 1.f / s;
    for (int t = tlead; t < tend; ++t) {  // pass 2: the run's rows are in L1 / L2 now
      const int slot = slots[t];
      if (slot < 0) continue;
      const int off = slot & (bs - 1);
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        if (lane + 32 * c < pieces) {
          const uint2 raw = reinterpret_cast<const uint2*>(kv + (int64_t)t * st + w * sw + h * sh)[lane + 32 * c];
          const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
          const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
          codes[off * pieces + lane + 32 * c] =
              encode4<E4M3>(clean(a.x) * inv, clean(a.y) * inv, clean(b.x) * inv, clean(b.y) * inv);
        }
      if (mass != nullptr && w == 0 && lane == 0) mass[(((int64_t)blk * Hk + h) << bs_log2) + off] = 0.f;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// bf16 copy of the listed blocks (exact: an 8-bit code times a power of two), for prompt attention,
// in blocks of 16 tokens whatever the cache's block size: dst [rows * mb16, 2, Hk, 16, D]. Row r of
// the table holds lens[r] tokens: what lies behind them reads as zero up to the next multiple
// of 128 tokens (the prompt kernels' KV tile) and is not written beyond it. 16 codes per thread.
// ---------------------------------------------------------------------------------------------
template <bool E4M3>
__global__ void __launch_bounds__(256)
    kv_dequant_scaled_kernel(const uint8_t* __restrict__ cache, const float* __restrict__ scales,
                             const int* __restrict__ tables, int64_t bt_stride, const int* __restrict__ lens, int mb16,
                             int num_blocks, int Hk, int D, int bs_log2, __nv_bfloat16* __restrict__ dst,
                             uint32_t* bounds) {
  const int r = blockIdx.y, i = blockIdx.x;             // table row, 16-token block of the row
  const int L = lens ? min(max(lens[r], 0), mb16 << 4) : mb16 << 4;
  const int tok0 = i << 4;
  if (tok0 >= ((L + 127) & ~127)) return;
  const int vec = D >> 4;                               // 16-code vectors per token row
  const int n = 2 * Hk * vec << 4;                      // of the destination block
  int64_t id = 0;
  if (tok0 < L) id = checked_index(tables[(int64_t)r * bt_stride + (tok0 >> bs_log2)], num_blocks, bounds);
  const int off0 = tok0 & ((1 << bs_log2) - 1);
  const int64_t out0 = ((int64_t)r * mb16 + i) * n;
  for (int v = threadIdx.x; v < n; v += 256) {
    const int rowi = v / vec;                           // (K/V, head, token)
    const int t = rowi & 15;
    uint4 o[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (tok0 + t < L) {
      const int64_t row = id * 2 * Hk + (rowi >> 4);
      const float s = scales[row];
      const uint4 c = reinterpret_cast<const uint4*>(cache)[((row << bs_log2) + off0 + t) * vec + v % vec];
      float f[16];
      decode4<E4M3>(c.x, f);
      decode4<E4M3>(c.y, f + 4);
      decode4<E4M3>(c.z, f + 8);
      decode4<E4M3>(c.w, f + 12);
#pragma unroll
      for (int k = 0; k < 16; ++k) f[k] *= s;
      o[0] = float_to_bf16x8(f);
      o[1] = float_to_bf16x8(f + 8);
    }
    uint4* d = reinterpret_cast<uint4*>(dst) + (out0 + v) * 2;
    d[0] = o[0];
    d[1] = o[1];
  }
}

// ---------------------------------------------------------------------------------------------
// Decode attention.
//
// One CTA takes a range of 16-token tiles of one (sequence, kv head); its 8 warps take the tiles in
// turn, each with its own ring of cp.async stages in shared memory, so no barrier stands in the loop. Heads are the
// N = 8 columns of mma.m16n8k16 and tokens (for S^T = K Q^T) or dims (for O^T = V^T P^T) the 16 rows, so a group of up
// to 8 heads wastes no row. Codes turn into f16 inside the fragments, exactly:
//   K: a lane's four consecutive bytes of a 16-byte chunk are two k-pairs of a k16 step. Any order of dims will
//      do as long as Q follows it, so Q is gathered in that order once.
//   V: ldmatrix.trans moves byte pairs; a byte permute splits them into the fragments of the even and the odd dims.
// Scores get the key scale, probabilities the value scale. The running reference m of the softmax
// covers score + exponent of the value scale, so p * scale fits f16 whatever the scales; the sum l
// uses p alone. m only moves when a score passes it by 2^8 (one vote per tile instead of a reduction).
// ---------------------------------------------------------------------------------------------
constexpr int kDecWarps = 8;
constexpr float kSlack = 8.f;  // p * scale <= 2^9: within f16

template <int D>
struct DecShape {
  static constexpr int kChunks = D / 16;                        // 16-byte chunks of a token row
  static constexpr int kRow = (kChunks | 1) * 16;               // row pitch: an odd number of chunks, so 8 rows of one chunk hit 8 bank groups
  static constexpr int kTile = 16 * kRow;
  static constexpr int kStage = 2 * kTile + 16;                 // K, V, two scales
  static constexpr int kStages = D <= 64 ? 4 : 3;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kCtas = D <= 128 ? 2 : 1;
};

struct DecArgs {
  const __nv_bfloat16* q;
  const uint8_t* cache;
  const float* scales;
  const int* tables;
  const int* lens;
  __nv_bfloat16* out;
  float* part_o;       // [B * H, splits, D]
  float* part_ml;      // [B * H, splits, 2]: reference (log2) and sum
  float* scores;       // [B * Hk, cap, G] log2 scores
  float* mass;
  int64_t q_stride, bt_stride;
  int B, H, Hk, G, NG, splits, mb, bs_log2, num_blocks, window;
  float scale_log2, cap, cap_log2;  // softcap (0: none): 2 / softcap, softcap * log2(e)
  uint32_t* bounds;
};

GOLLEK_DEVICE void cp_async16(uint32_t dst, const void* src, bool full) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
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
GOLLEK_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

template <int D, int NT, bool E4M3, bool MASS>
__global__ void __launch_bounds__(kDecWarps * 32, DecShape<D>::kCtas) block8_decode_kernel(const DecArgs p) {
  using S = DecShape<D>;
  constexpr int CH = S::kChunks, HB = 8 * NT;  // heads of this CTA
  extern __shared__ __align__(16) uint8_t dsm[];
  __shared__ float sm_m[kDecWarps][HB], sm_l[kDecWarps][HB];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  int idx = blockIdx.x;
  const int split = idx % p.splits;
  idx /= p.splits;
  const int hg = idx % p.NG;
  const int bk = idx / p.NG;  // b * Hk + kh
  const int kh = bk % p.Hk, b = bk / p.Hk;
  const int h0 = hg * HB, nh = min(p.G - h0, HB);  // heads of the group handled here
  const int L = min(max(p.lens[b], 0), p.mb << p.bs_log2);
  const int lo = p.window > 0 ? max(0, L - p.window) : 0;
  const int t_lo = lo >> 4, t_hi = (L + 15) >> 4;
  const int per = (t_hi - t_lo + p.splits - 1) / p.splits;
  const int tb = t_lo + split * per, te = min(t_hi, tb + per);
  const int mine = tb + warp < te ? (te - tb - warp + kDecWarps - 1) / kDecWarps : 0;
  const int* bt = p.tables + (int64_t)b * p.bt_stride;
  uint8_t* ring = dsm + warp * S::kRing;
  const uint32_t ring_u = smem_u32(ring);

  int ids = 0;  // lane l: pool block of this warp's tile (j & ~31) + l
  auto issue = [&](int j) {
    if (j < mine) {
      if ((j & 31) == 0) {
        const int t = tb + warp + kDecWarps * (j + lane);
        ids = t < te ? checked_index(bt[t >> (p.bs_log2 - 4)], p.num_blocks, p.bounds) : 0;
      }
      const int64_t id = __shfl_sync(0xffffffffu, ids, j & 31);
      const int t = tb + warp + kDecWarps * j;
      const int off = (t << 4) & ((1 << p.bs_log2) - 1);
      const int64_t rk = (id * 2) * p.Hk + kh, rv = rk + p.Hk;
      const uint8_t* gk = p.cache + ((rk << p.bs_log2) + off) * D;
      const uint8_t* gv = p.cache + ((rv << p.bs_log2) + off) * D;
      const uint32_t st = ring_u + (j % S::kStages) * S::kStage;
#pragma unroll
      for (int i = 0; i < CH / 2; ++i) {
        const int e = i * 32 + lane, row = e / CH, ch = e % CH;
        const int tok = (t << 4) + row;
        const bool full = tok >= lo && tok < L;  // rows outside read as zero
        cp_async16(st + row * S::kRow + ch * 16, gk + e * 16, full);
        cp_async16(st + S::kTile + row * S::kRow + ch * 16, gv + e * 16, full);
      }
      if (lane < 2) cp_async4(st + 2 * S::kTile + 4 * lane, p.scales + (lane ? rv : rk));
    }
    cp_async_commit();
  };
#pragma unroll
  for (int j = 0; j < S::kStages - 1; ++j) issue(j);

  // Q^T as the B operand, columns = heads: chunk j of the lane's head, dims 16 j + 4 c + {0, 1} and
  // + {2, 3}. Each head is brought to an amax in [2^11, 2^12) by a power of two: f16 then holds every
  // bf16 within 2^-28 of it exactly.
  uint32_t qf[NT][CH][2];
  float qmul[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int hh = nt * 8 + g;
    uint2 raw[CH];
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      raw[j] = make_uint2(0u, 0u);
      if (hh < nh)
        raw[j] = *reinterpret_cast<const uint2*>(p.q + (int64_t)b * p.q_stride + (int64_t)(kh * p.G + h0 + hh) * D + 16 * j + 4 * c);
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[j].x));
      const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[j].y));
      amax = fmaxf(amax, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 127) - 11;
    const float f = __uint_as_float((uint32_t)(127 - e) << 23);
    const float back = __uint_as_float((uint32_t)(127 + e) << 23) * p.scale_log2;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[j].x));
      const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[j].y));
      const __half2 hx = __floats2half2_rn(x.x * f, x.y * f), hy = __floats2half2_rn(y.x * f, y.y * f);
      qf[nt][j][0] = *reinterpret_cast<const uint32_t*>(&hx);
      qf[nt][j][1] = *reinterpret_cast<const uint32_t*>(&hy);
    }
    qmul[nt][0] = __shfl_sync(0xffffffffu, back, 8 * c);      // columns 2 c and 2 c + 1
    qmul[nt][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
  }

  float o[CH][NT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int j = 0; j < CH; ++j)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][nt][e] = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;

  // ldmatrix row of this lane: matrices (rows 0-7, 8-15) of one chunk, then of the next
  const uint32_t ld_off = ((lane & 7) + ((lane >> 3) & 1) * 8) * S::kRow + (lane >> 4) * 16;
  for (int j = 0; j < mine; ++j) {
    cp_async_wait<S::kStages - 2>();
    __syncwarp();
    issue(j + S::kStages - 1);  // into the stage read in the previous turn
    const uint32_t st = ring_u + (j % S::kStages) * S::kStage;
    float s[NT][4], s2[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][e] = 0.f;
#pragma unroll
    for (int j2 = 0; j2 < CH / 2; ++j2) {
      uint32_t r[4], a[4];
      ldsm4(r, st + ld_off + j2 * 32);
      expand4<E4M3, false>(r[0], a[0], a[2]);
      expand4<E4M3, false>(r[1], a[1], a[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a, qf[nt][2 * j2][0], qf[nt][2 * j2][1]);
      expand4<E4M3, false>(r[2], a[0], a[2]);
      expand4<E4M3, false>(r[3], a[1], a[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16(s2[nt], a, qf[nt][2 * j2 + 1][0], qf[nt][2 * j2 + 1][1]);
    }
    float ks, vs;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(ks), "=f"(vs) : "r"(st + 2 * S::kTile) : "memory");
    const float ev = (float)max((int)((__float_as_uint(vs) >> 23) & 0xff) - 127, -100);
    const int tok = ((tb + warp + kDecWarps * j) << 4) + g;
    const bool ok0 = tok >= lo && tok < L, ok1 = tok + 8 >= lo && tok + 8 < L;
    bool up = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = (s[nt][e] + s2[nt][e]) * (ks * qmul[nt][e & 1]);
        // cap * tanh(x / cap) = cap * (1 - 2 / (1 + e^(2 x / cap)))
        if (p.cap > 0.f) x = p.cap_log2 * (1.f - __fdividef(2.f, 1.f + ex2(x * p.cap)));
        s[nt][e] = (e < 2 ? ok0 : ok1) ? x : -INFINITY;
        up |= s[nt][e] + ev > m[nt][e & 1] + kSlack;
      }
    if constexpr (MASS) {
      float* sc = p.scores + ((int64_t)bk * (p.mb << p.bs_log2) + tok) * p.G + h0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int hh = nt * 8 + 2 * c + (e & 1);
          if (hh < nh && (e < 2 ? ok0 : ok1)) sc[(e < 2 ? 0 : 8 * p.G) + hh] = s[nt][e];
        }
    }
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[nt][e], s[nt][e + 2]) + ev;
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          x = fmaxf(x, m[nt][e]);
          const float d = x > m[nt][e] ? m[nt][e] - x : 0.f, al = ex2(d);
          m[nt][e] = x;
          l[nt][e] = shift_sum(l[nt][e], d);
#pragma unroll
          for (int jj = 0; jj < CH; ++jj) o[jj][nt][e] *= al, o[jj][nt][e + 2] *= al;
        }
    }
    uint32_t pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float e0 = ok0 ? ex2(s[nt][0] - m[nt][0]) : 0.f, e1 = ok0 ? ex2(s[nt][1] - m[nt][1]) : 0.f;
      float e2 = ok1 ? ex2(s[nt][2] - m[nt][0]) : 0.f, e3 = ok1 ? ex2(s[nt][3] - m[nt][1]) : 0.f;
      l[nt][0] += e0 + e2;
      l[nt][1] += e1 + e3;
      // probabilities in f16 (2^-11 relative): the output's bf16 rounding is eight times coarser
      const __half2 x = __floats2half2_rn(e0 * vs, e1 * vs), y = __floats2half2_rn(e2 * vs, e3 * vs);
      pb[nt][0] = movm_t(*reinterpret_cast<const uint32_t*>(&x));
      pb[nt][1] = movm_t(*reinterpret_cast<const uint32_t*>(&y));
    }
#pragma unroll
    for (int j2 = 0; j2 < CH / 2; ++j2) {
      uint32_t r[4], a[4];
      ldsm4_t(r, st + S::kTile + ld_off + j2 * 32);
      expand4<E4M3, true>(r[0], a[0], a[1]);
      expand4<E4M3, true>(r[1], a[2], a[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16(o[2 * j2][nt], a, pb[nt][0], pb[nt][1]);
      expand4<E4M3, true>(r[2], a[0], a[1]);
      expand4<E4M3, true>(r[3], a[2], a[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16(o[2 * j2 + 1][nt], a, pb[nt][0], pb[nt][1]);
    }
  }
  cp_async_wait<0>();
  __syncwarp();

  // the warps' partial sums meet in shared memory (each over its own ring)
  static_assert(HB * D * 4 <= S::kRing, "a warp's partial output fits its ring");
  float* wo = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int hh = nt * 8 + 2 * c + e;
      float x = l[nt][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) sm_m[warp][hh] = m[nt][e], sm_l[warp][hh] = x;
#pragma unroll
      for (int j = 0; j < CH; ++j)
        *reinterpret_cast<float2*>(wo + hh * D + 16 * j + 2 * g) = make_float2(o[j][nt][e], o[j][nt][e + 2]);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < nh * D; i += kDecWarps * 32) {
    const int hh = i / D;
    float M = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sm_m[w][hh]);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float d = sm_m[w][hh] - M, f = sm_m[w][hh] == -INFINITY ? 0.f : ex2(d);
      if (sm_m[w][hh] != -INFINITY) sum += shift_sum(sm_l[w][hh], d);
      acc += f * reinterpret_cast<const float*>(dsm + w * S::kRing)[i];
    }
    const int64_t row = (int64_t)b * p.H + kh * p.G + h0 + hh;
    if (p.splits == 1)
      p.out[row * D + i % D] = __float2bfloat16(sum > 0.f ? acc / sum : 0.f);
    else
      p.part_o[(row * p.splits + split) * D + i % D] = acc;
    if ((p.splits > 1 || MASS) && i % D == 0)
      *reinterpret_cast<float2*>(p.part_ml + (row * p.splits + split) * 2) = make_float2(M, sum);
  }
}

// Joins the splits of each (sequence, head): the first B * H CTAs; the others add the softmax weights
// of 256 tokens of a (sequence, kv head) to mass, summed over the head group in head order. An entry gets one add
// per call, so sums do not depend on the order of the CTAs unless sequences share a block.
__global__ void __launch_bounds__(128) block8_join_kernel(const DecArgs p, int D, int mass_tiles) {
  __shared__ float sm[128];
  const int joins = p.splits > 1 ? p.B * p.H : 0;
  if ((int)blockIdx.x < joins) {
    const int64_t row = blockIdx.x;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row * p.splits;
    float M = -INFINITY, sum = 0.f;
    for (int i = 0; i < p.splits; ++i) M = fmaxf(M, ml[i].x);
    for (int i = 0; i < p.splits; ++i) sum += ml[i].x == -INFINITY ? 0.f : shift_sum(ml[i].y, ml[i].x - M);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    for (int d = threadIdx.x; d < D; d += 128) {
      float acc = 0.f;
      for (int i = 0; i < p.splits; ++i)
        if (ml[i].x != -INFINITY) acc += ex2(ml[i].x - M) * p.part_o[(row * p.splits + i) * D + d];
      p.out[row * D + d] = __float2bfloat16(acc * inv);
    }
    return;
  }
  const int i = blockIdx.x - joins;
  const int bk = i / mass_tiles, kh = bk % p.Hk, b = bk / p.Hk;
  const int L = min(max(p.lens[b], 0), p.mb << p.bs_log2);
  const int lo = p.window > 0 ? max(0, L - p.window) : 0;
  const int first = (i % mass_tiles) * 256;
  if (first >= L || first + 256 <= lo) return;
  for (int h = threadIdx.x; h < p.G; h += 128) {
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + ((int64_t)b * p.H + kh * p.G + h) * p.splits;
    float M = -INFINITY, sum = 0.f;
    for (int k = 0; k < p.splits; ++k) M = fmaxf(M, ml[k].x);
    for (int k = 0; k < p.splits; ++k) sum += ml[k].x == -INFINITY ? 0.f : shift_sum(ml[k].y, ml[k].x - M);
    sm[h] = M + log2f(sum);
  }
  __syncthreads();
  for (int t = first + threadIdx.x; t < min(first + 256, L); t += 128) {
    if (t < lo) continue;
    const float* sc = p.scores + ((int64_t)bk * (p.mb << p.bs_log2) + t) * p.G;
    float w = 0.f;
    for (int h = 0; h < p.G; ++h) w += ex2(sc[h] - sm[h]);
    const int64_t id = checked_index(p.tables[(int64_t)b * p.bt_stride + (t >> p.bs_log2)], p.num_blocks, p.bounds);
    atomicAdd(p.mass + ((id * p.Hk + kh) << p.bs_log2) + (t & ((1 << p.bs_log2) - 1)), w);
  }
}

// ---------------------------------------------------------------------------------------------
// Eviction, step 1: which tokens stay. One CTA per (layer, sequence, kv head).
//
// Of a sequence with L tokens and K < L to keep: the first a = min(sink, K), the last
// r = min(recent, K - a), and of those between the K - a - r with the largest mass (ties: the lower
// index). A radix select (11 + 11 + 10 bits of the order-preserving integer of the mass) finds the
// smallest mass that stays and how many tokens of exactly that mass do; one ordered pass lists them.
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
  // prefix is the smallest key that stays, `want` how many tokens with it do (the first ones)
  uint32_t gt0 = 0, eq0 = 0;
  for (int base = 0; base < n; base += kSelThreads) {
    const int i = base + threadIdx.x;
    const uint32_t k = i < n ? (held ? keys[i] : load(i)) : 0u;
    const uint32_t gt = i < n && k > prefix, eq = i < n && k == prefix;
    uint32_t total;
    const uint32_t before = block_scan((gt << 16) | eq, warp_sums, total);
    const uint32_t gb = gt0 + (before >> 16), eb = eq0 + (before & 0xffffu);
    if (gt || (eq && eb < want)) kept[a + gb + min(eb, want)] = c0 + i;
    gt0 += total >> 16;
    eq0 += total & 0xffffu;
  }
}

// ---------------------------------------------------------------------------------------------
// Eviction, step 2: the kept tokens move to the front, in order. One CTA per (layer, sequence, kv head, K/V).
//
// In place: kept[j] >= j, so a chunk's sources lie at or behind its own places and every chunk that is
// overwritten by it has been read (chunks go up, a chunk's loads end before its stores). Each destination block
// gets the smallest power-of-two scale for what it then holds.
// ---------------------------------------------------------------------------------------------
constexpr int kMoveThreads = 256;

template <bool E4M3>
__global__ void __launch_bounds__(kMoveThreads) kv_evict_move_kernel(const EvictArgs p) {
  constexpr int kItems = 4;       // 16-byte pieces per thread and chunk
  __shared__ uint32_t top[64];    // largest magnitude of each destination block of the chunk (float bits)
  const int h = blockIdx.x >> 1, w = blockIdx.x & 1, b = blockIdx.y, ly = blockIdx.z;
  const EvictRow r = evict_row(p, b);
  if (!r.cut || r.K == 0) return;
  const int bs = 1 << p.bs_log2, vec = p.D >> 4;
  const int chunk = kMoveThreads * kItems / vec / 64 * 64;  // tokens, a multiple of every block size
  const int* kept = p.kept + (((int64_t)ly * p.B + b) * p.Hk + h) * p.max_keep;
  const int* bt = p.tables + (int64_t)b * p.bt_stride;
  const int64_t pool = (int64_t)ly * p.num_blocks;
  auto row_of = [&](int t) {  // (block, K/V, head) row of token t's block
    const int64_t id = pool + checked_index(bt[t >> p.bs_log2], p.num_blocks, p.bounds);
    return (id * 2 + w) * p.Hk + h;
  };
  auto mass_at = [&](int t) {
    const int64_t id = pool + checked_index(bt[t >> p.bs_log2], p.num_blocks, p.bounds);
    return p.mass + ((id * p.Hk + h) << p.bs_log2) + (t & (bs - 1));
  };
  for (int base = 0; base < r.K; base += chunk) {
    const int n = min(chunk, r.K - base);
    if (threadIdx.x < 64) top[threadIdx.x] = 0u;
    __syncthreads();
    uint4 code[kItems];
    float sc[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int e = k * kMoveThreads + threadIdx.x, j = e / vec;
      sc[k] = 0.f;
      if (j < n) {
        const int t = kept[base + j];
        const int64_t row = row_of(t);
        code[k] = *reinterpret_cast<const uint4*>(p.cache + ((row << p.bs_log2) + (t & (bs - 1))) * p.D + (e % vec) * 16);
        sc[k] = p.scales[row];
      }
    }
    float mv[2];  // masses travel with the K pass (chunk <= 2 * kMoveThreads)
    if (w == 0)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (k * kMoveThreads + (int)threadIdx.x < n) mv[k] = *mass_at(kept[base + k * kMoveThreads + threadIdx.x]);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int j = (k * kMoveThreads + threadIdx.x) / vec;
      if (j < n) {
        float f[16], amax = 0.f;
        decode4<E4M3>(code[k].x, f);
        decode4<E4M3>(code[k].y, f + 4);
        decode4<E4M3>(code[k].z, f + 8);
        decode4<E4M3>(code[k].w, f + 12);
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(f[i]));
        atomicMax(&top[j >> p.bs_log2], __float_as_uint(amax * sc[k]));
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int e = k * kMoveThreads + threadIdx.x, j = e / vec;
      if (j < n) {
        const int to = base + j;
        const float s = pow2_scale<E4M3>(__uint_as_float(top[j >> p.bs_log2]));
        const float ratio = sc[k] / s;
        const int64_t row = row_of(to);
        float f[16];
        decode4<E4M3>(code[k].x, f);
        decode4<E4M3>(code[k].y, f + 4);
        decode4<E4M3>(code[k].z, f + 8);
        decode4<E4M3>(code[k].w, f + 12);
        uint4 o;
        o.x = encode4<E4M3>(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
        o.y = encode4<E4M3>(f[4] * ratio, f[5] * ratio, f[6] * ratio, f[7] * ratio);
        o.z = encode4<E4M3>(f[8] * ratio, f[9] * ratio, f[10] * ratio, f[11] * ratio);
        o.w = encode4<E4M3>(f[12] * ratio, f[13] * ratio, f[14] * ratio, f[15] * ratio);
        *reinterpret_cast<uint4*>(p.cache + ((row << p.bs_log2) + (to & (bs - 1))) * p.D + (e % vec) * 16) = o;
        if ((to & (bs - 1)) == 0 && e % vec == 0) p.scales[row] = s;
      }
    }
    if (w == 0)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (k * kMoveThreads + (int)threadIdx.x < n) *mass_at(base + k * kMoveThreads + threadIdx.x) = mv[k];
    __syncthreads();
  }
}

int log2_block(int bs) {
  throw_if(bs != 16 && bs != 32 && bs != 64, "block-scaled KV cache: block size 16, 32 or 64");
  return bs == 16 ? 4 : bs == 32 ? 5 : 6;
}

}  // namespace

void launch_kv_quant_blocks(const void* kv, int64_t st, int64_t sw, int64_t sh, const int* slots, void* cache,
                            float* scales, float* mass, int T, int Hk, int D, int bs, int num_blocks, bool e4m3,
                            cudaStream_t s) {
  throw_if(D % 4 != 0 || D > 256, "block-scaled KV cache: head_dim must be a multiple of 4, <= 256");
  const int lb = log2_block(bs);
  if (T == 0) return;
  const int g = T >= 1024 ? 16 : 1;  // tokens a warp looks at: about one run of a prompt, one row of a decode step
  const int64_t warps = (int64_t)((T + g - 1) / g) * 2 * Hk;
  const unsigned grid = (unsigned)((warps + 7) / 8);
#define GOLLEK_QB(E, N)                                                                                              \
  kv_quant_blocks_kernel<E, N><<<grid, 256, 0, s>>>(reinterpret_cast<const __nv_bfloat16*>(kv), st, sw, sh, slots,    \
                                                    reinterpret_cast<uint8_t*>(cache), scales, mass, T, Hk, D, lb,    \
                                                    num_blocks, g, bounds_status())
  if (D <= 128) {
    if (e4m3) GOLLEK_QB(true, 1);
    else GOLLEK_QB(false, 1);
  } else {
    if (e4m3) GOLLEK_QB(true, 2);
    else GOLLEK_QB(false, 2);
  }
#undef GOLLEK_QB
  check_launch("kv_quant_blocks");
}

void launch_kv_dequant_scaled(const void* cache, const float* scales, const int* tables, int64_t bt_stride,
                              const int* lens, int rows, int mb, int num_blocks, int Hk, int D, int bs, bool e4m3,
                              void* dst, cudaStream_t s) {
  throw_if(D % 16 != 0, "block-scaled KV cache: head_dim must be a multiple of 16");
  const int lb = log2_block(bs);
  throw_if(rows > 65535, "kv_dequant_blocks: at most 65535 sequences");
  if (rows == 0 || mb == 0) return;
  auto k = e4m3 ? kv_dequant_scaled_kernel<true> : kv_dequant_scaled_kernel<false>;
  const int mb16 = mb << (lb - 4);
  k<<<dim3(mb16, rows), 256, 0, s>>>(reinterpret_cast<const uint8_t*>(cache), scales, tables, bt_stride, lens, mb16,
                                     num_blocks, Hk, D, lb, reinterpret_cast<__nv_bfloat16*>(dst), bounds_status());
  check_launch("kv_dequant_blocks");
}

// Splits of each (sequence, kv head): enough CTAs for two rounds of the GPU, at least 16 tiles (256
// tokens) each, as far as the table's width says.
int block8_decode_splits(int B, int Hk, int G, int D, int64_t max_len) {
  const int nt = (G > 8 && D <= 128) ? 2 : 1, ng = (G + 8 * nt - 1) / (8 * nt);
  const int64_t ctas = (int64_t)B * Hk * ng;
  const int64_t slots = (int64_t)device_num_sms() * (D <= 128 ? 2 : 1);
  if (ctas == 0 || ctas >= 2 * slots) return 1;
  const int64_t want = (2 * slots + ctas - 1) / ctas;
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(want, (max_len + 255) / 256), 64));
}

void launch_block8_decode(void* out, const void* q, int64_t q_stride, const void* cache, const float* scales,
                          const int* tables, int64_t bt_stride, int mb, const int* lens, int B, int H, int Hk, int D,
                          int bs, int num_blocks, int splits, float scale, int window, float softcap, float* part_o,
                          float* part_ml, float* scores, float* mass, bool e4m3, cudaStream_t s) {
  DecArgs p;
  p.bs_log2 = log2_block(bs);
  if (B == 0) return;
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.cache = reinterpret_cast<const uint8_t*>(cache);
  p.scales = scales;
  p.tables = tables;
  p.lens = lens;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.part_o = part_o;
  p.part_ml = part_ml;
  p.scores = scores;
  p.mass = mass;
  p.q_stride = q_stride;
  p.bt_stride = bt_stride;
  p.B = B, p.H = H, p.Hk = Hk, p.G = H / Hk, p.splits = splits, p.mb = mb, p.num_blocks = num_blocks, p.window = window;
  const int nt = (p.G > 8 && D <= 128) ? 2 : 1;  // D = 256: two column tiles would need 128 accumulators a lane
  p.NG = (p.G + 8 * nt - 1) / (8 * nt);
  p.scale_log2 = scale * kLog2e;
  p.cap = softcap > 0.f ? 2.f / softcap : 0.f;  // scores are in log2 units: e^(2 x / cap) = 2^(2 x log2(e) / cap)
  p.cap_log2 = softcap * kLog2e;
  p.bounds = bounds_status();
  throw_if(p.G > 128, "block-scaled decode attention: at most 128 query heads per KV head");
  const int64_t grid = (int64_t)B * Hk * p.NG * splits;
  throw_if(grid > 0x7fffffff, "block-scaled decode attention: grid too large");
  bool done = false;
  auto go = [&](auto kern, int smem) {
    GOLLEK_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kern<<<(unsigned)grid, kDecWarps * 32, smem, s>>>(p);
    done = true;
  };
#define GOLLEK_B8_M(DD, NN, M)                                                          \
  if (e4m3) go(block8_decode_kernel<DD, NN, true, M>, kDecWarps * DecShape<DD>::kRing); \
  else go(block8_decode_kernel<DD, NN, false, M>, kDecWarps * DecShape<DD>::kRing)
#define GOLLEK_B8_N(DD, NN) \
  if (mass) { GOLLEK_B8_M(DD, NN, true); } else { GOLLEK_B8_M(DD, NN, false); }
#define GOLLEK_B8(DD) \
  if (D == DD) {      \
    if (nt == 1) { GOLLEK_B8_N(DD, 1) } else { GOLLEK_B8_N(DD, 2) } \
  }
  GOLLEK_B8(32)
  GOLLEK_B8(64)
  GOLLEK_B8(96)
  GOLLEK_B8(128)
  if (D == 256) { GOLLEK_B8_N(256, 1) }
#undef GOLLEK_B8
#undef GOLLEK_B8_N
#undef GOLLEK_B8_M
  throw_if(!done, "block-scaled decode attention: unsupported head_dim " + std::to_string(D));
  check_launch("block8_decode");
  const int mass_tiles = mass ? ((mb << p.bs_log2) + 255) / 256 : 0;
  const int64_t join = (splits > 1 ? (int64_t)B * H : 0) + (int64_t)B * Hk * mass_tiles;
  throw_if(join > 0x7fffffff, "block-scaled decode attention: grid too large");
  if (join > 0) {
    block8_join_kernel<<<(unsigned)join, 128, 0, s>>>(p, D, mass_tiles);
    check_launch("block8_join");
  }
}

void launch_kv_evict(void* cache, float* scales, float* mass, const int* tables, int64_t bt_stride, int mb,
                     const int* lens, const int* keep, int* kept, int layers, int B, int Hk, int D, int bs,
                     int num_blocks, int sink, int recent, int max_keep, bool e4m3, cudaStream_t s) {
  throw_if(D % 16 != 0 || D < 32 || D > 256, "kv_evict: head_dim must be a multiple of 16, 32 to 256");
  throw_if(B > 65535 || layers > 65535, "kv_evict: at most 65535 sequences and layers");
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
  GOLLEK_CUDA_CHECK(cudaFuncSetAttribute(kv_evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelKeys * 4));
  kv_evict_select_kernel<<<dim3(Hk, B, layers), kSelThreads, smem, s>>>(p);
  check_launch("kv_evict_select");
  if (max_keep == 0) return;
  auto k = e4m3 ? kv_evict_move_kernel<true> : kv_evict_move_kernel<false>;
  k<<<dim3(2 * Hk, B, layers), kMoveThreads, 0, s>>>(p);
  check_launch("kv_evict_move");
}

}  // namespace gollek
