// The 4-bit KV cache format and the warp-level tile arithmetic over it.
//
// One layer's cache is uint8 [pages, Hkv, page size / 16, 2 (K, V), record].
// A record holds 16 tokens of one head: 1024 bytes of 4-bit codes, then per
// group of G channels (32, 64 or 128) 16 words, one per token, of
// (bf16 scale << 16 | fp16 zero point). Code c of scale s and zero point z
// stands for s * (c + z):
//
//   lo = min(0, min x)   hi = max(0, max x)   s = bf16((hi - lo) / 15)
//   z = fp16(lo / s) in [-15.1, 0]            c = clamp(rint(x / s - z), 0, 15)
//
// over the group's inputs, which saturate at +-8192 (a NaN counts as 0); a
// group whose step is below 2^-120 is stored as zeros. The limit keeps s below
// 2^10.1; the scale is bf16 so that small groups keep their relative precision
// (the kernels take a power of two out of it before anything becomes fp16).
//
// Order of the codes. The matrix instruction m16n8k16 takes its A operand as
// 16-bit pairs; a 32-bit word of 8 codes gives four pairs by masking, because
// the code at bits 0-3 (or 4-7) of a half is the fp16 subnormal c * 2^-24
// (c * 2^-20), exactly. With g = lane / 4, t = lane % 4:
//   K: token r's 64 bytes; word 4 t + i holds channels 32 i + 8 t + 0..7 in
//      nibble order, so one 16-byte load of lane (r % 8, t) is A for all eight
//      k-steps (32 channels per word index i).
//   V: word 128 (m / 4) + 4 lane + m % 4 is lane's A fragment of the transposed
//      16 channel x 16 token tile m: nibble (ch / 8 % 2) + 2 (tok / 8) +
//      4 (tok % 2) of channel 16 m + 8 (ch / 8 % 2) + g, token
//      8 (tok / 8) + 2 t + tok % 2. A byte belongs to one token, so single
//      tokens are written without a read.
#pragma once
#include <cuda_fp16.h>

#include "attn_common.cuh"

namespace dsv {

constexpr int KV4_CODES = 1024;           // bytes of codes of a record (16 tokens x 128 channels)
constexpr float KV4_LIMIT = 8192.f;
constexpr float KV4_TINY = 7.52316385e-37f;  // 2^-120

__host__ __device__ constexpr int kv4_record(int ng) { return KV4_CODES + 64 * ng; }

__device__ __forceinline__ float kv4_scale(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float kv4_zero(uint32_t w) {
  return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu)));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Transpose of an 8 x 8 tile of 16-bit values held as an MMA fragment.
__device__ __forceinline__ uint32_t movm_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ void cp_async4(void* smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}

__device__ __forceinline__ float kv4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Bounded wait as mbar_wait, but for two things: it polls a while before its
// limit's clock is read (these kernels' stages turn over in well under a
// microsecond), and a recorded kErrShape does not end it. That one says that an
// index of some call was out of range and not followed; the waits still complete,
// and the other sequences their results.
__device__ __forceinline__ bool kv4_wait(uint64_t* bar, uint32_t parity, int code) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t n = 1;; ++n) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((n & 1023u) == 0) {
      const int seen = *(volatile int*)&g_error;
      if (seen != 0 && seen != kErrShape) return false;
      if (globaltimer_ns() - t0 > kWaitNs) {
        if (seen != 0) atomicCAS(&g_error, kErrShape, code);
        else set_error(code);
        return false;
      }
    }
  }
}

// Bounded wait that goes on when another wait has given up: for what must end
// before shared or tensor memory is given back.
__device__ __forceinline__ void kv4_drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - t0 < kWaitNs) {
  }
}

// Online softmax attention of up to 8 * NH query columns (a column = one query
// head) over 16-token records, one warp. Per column the weights are
// p = 2^(score - m + 2) against a reference maximum m that moves only when a
// score exceeds it by more than 3 (base-2 units): p stays below 2^5 and the
// common factor cancels in O / l.
//
// Scores: S = sum_groups s (q . c) + s z sum(q): the codes enter the matrix
// instruction as fp16 subnormals and the query as fp16 scaled by a power of two
// per column (its largest magnitude lands in [2^14, 2^15); bf16 fits fp16's
// mantissa, so this is exact down to 2^-29 of the largest), and the products
// are undone by `f`. Output: O = sum w c + sum w z with w = p s 2^-r rounded to
// fp16 (11 bits), the second sum one fp32 number per group and column. Both sums
// take the rounded w, so that a weight's rounding scales its key's value as a
// whole. Each group of channels has its own power of two, r: it puts the group's
// largest scale into [2^7, 2^8) and moves, as the reference maximum does, when one
// of 2^10 or more comes. So w stays below 2^15, and a key keeps its 11 bits down
// to 2^-23 of the largest p s of its group, whatever the values' size (a fixed r
// lost small groups altogether, and the small weights beside a dominant key: 4 %
// of the result for values near 1e-6).
constexpr float KV4_P_BIAS = 2.f;
constexpr float KV4_LAZY = 3.f;
constexpr int KV4_R_TOP = 7;
constexpr uint32_t KV4_R_SUM = (127u + KV4_R_TOP + 127 + 3) << 23;   // bits of 2^-r plus those of the scale that moves it
constexpr int KV4_R_MIN = -110;              // exponent of the smallest scale that r follows: 2^-r stays finite

template <int NG, int NH>
struct Kv4Warp {
  uint32_t q[NH][8][2];   // B fragments of the query, k-step by k-step
  float f[NH][2];         // score factor of columns 2t, 2t + 1
  float qs[NH][NG][2];    // scaled sum of the query over each group
  float acc[NH][8][4];    // sum p s c, channels 16 m + g (+ 8: times 16) x columns 2t, 2t + 1; times 2^-24
  float z[NH][NG][2];     // this lane's share of sum w z
  float* rs;              // 2^-r of each group, in shared memory: registers are short
  float m[NH][2], l[NH][2];
  float ref[NH][2];       // what scores are taken against: m - KV4_P_BIAS, 0 before the first

  // `row(h)` gives the address of column h's 128 query values, null past the last one.
  template <class Row>
  __device__ __forceinline__ void begin(Row row, float scale_log2) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      uint32_t x[4][4];                     // 8 channels 32 i + 8 t + 0..7 of column 8 n + g each
      const __nv_bfloat16* src = row(n * 8 + g);
      __nv_bfloat162 top = __float2bfloat162_rn(0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (src != nullptr) w = *reinterpret_cast<const uint4*>(src + 32 * i + 8 * t);
        x[i][0] = w.x;
        x[i][1] = w.y;
        x[i][2] = w.z;
        x[i][3] = w.w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&x[i][e])));
      float amax = fmaxf(__low2float(top), __high2float(top));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // amax in [2^e, 2^(e+1)): scale by 2^(14 - e), e kept where that is a normal float
      const int e = min(127, max(-100, (int)((__float_as_uint(amax) >> 23) & 255u) - 127));
      const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
      const float down = up * 0.0625f;
      const float fh = scale_log2 * __uint_as_float((uint32_t)min(254, 127 + e + 10) << 23);   // 2^24 / up
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          v[2 * c] = __uint_as_float(x[i][c] << 16);
          v[2 * c + 1] = __uint_as_float(x[i][c] & 0xffff0000u);
        }
        q[n][2 * i][0] = pack_f16(v[0] * up, v[4] * up);
        q[n][2 * i][1] = pack_f16(v[1] * down, v[5] * down);
        q[n][2 * i + 1][0] = pack_f16(v[2] * up, v[6] * up);
        q[n][2 * i + 1][1] = pack_f16(v[3] * down, v[7] * down);
      }
      // the scores' columns are 2t, 2t + 1: fetch those columns' factors
      f[n][0] = __shfl_sync(0xffffffffu, fh, 8 * t);
      f[n][1] = __shfl_sync(0xffffffffu, fh, 8 * t + 4);
      // sums over the groups by the same products, with ones (and 16 for the lowered half) for codes
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8 / NG; ++k)
          mma_f16(d, 0x3c003c00u, 0x3c003c00u, 0x4c004c00u, 0x4c004c00u, q[n][i * (8 / NG) + k][0],
                  q[n][i * (8 / NG) + k][1]);
        qs[n][i][0] = f[n][0] * 5.9604644775390625e-8f * d[0];   // 2^-24
        qs[n][i][1] = f[n][1] * 5.9604644775390625e-8f * d[1];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[n][c] = -INFINITY;
        l[n][c] = ref[n][c] = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) z[n][i][c] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
    }
    __syncwarp();                            // the last segment's readers are done
#pragma unroll
    for (int i = 0; i < NG; ++i)
      if (lane == 0) rs[i] = __uint_as_float((uint32_t)(127 + KV4_R_TOP - KV4_R_MIN) << 23);
    __syncwarp();
  }

  // Two K and V records (32 tokens; 16-byte aligned), of which the first `valid`
  // tokens are seen. An unseen token's weight is 0 whatever its record holds.
  __device__ __forceinline__ void tokens(const uint8_t* rec, int valid) {
    if (valid >= 32) tokens_of<true>(rec, 32);
    else tokens_of<false>(rec, valid);
  }
  template <bool ALL>
  __device__ __forceinline__ void tokens_of(const uint8_t* rec, int valid) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int KREC = kv4_record(NG);
    float s[NH][8];                         // element 4 r + 2 i + c: token 16 r + 8 i + g, column 8 n + 2 t + c
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* krec = rec + r * 2 * KREC;
      const uint4 k0 = *reinterpret_cast<const uint4*>(krec + 16 * lane);
      const uint4 k1 = *reinterpret_cast<const uint4*>(krec + 512 + 16 * lane);
      const uint32_t kw0[4] = {k0.x, k0.y, k0.z, k0.w}, kw1[4] = {k1.x, k1.y, k1.z, k1.w};
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(krec + KV4_CODES) + g;
      float zq[NH][4];
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        float d[NH][4];
#pragma unroll
        for (int n = 0; n < NH; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.f;
#pragma unroll
        for (int j = 0; j < 4 / NG; ++j) {
          const int i = ng * (4 / NG) + j;
          const uint32_t w0 = kw0[i], w1 = kw1[i], x0 = w0 >> 8, x1 = w1 >> 8;
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            mma_f16(d[n], w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, q[n][2 * i][0],
                    q[n][2 * i][1]);
            mma_f16(d[n], x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u, q[n][2 * i + 1][0],
                    q[n][2 * i + 1][1]);
          }
        }
        const uint32_t p0 = kp[ng * 16], p1 = kp[ng * 16 + 8];
        const float s0 = kv4_scale(p0), s1 = kv4_scale(p1);
        const float b0 = s0 * kv4_zero(p0), b1 = s1 * kv4_zero(p1);
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float* v = &s[n][4 * r + c];
            v[0] = ng == 0 ? s0 * d[n][c] : fmaf(s0, d[n][c], v[0]);
            v[2] = ng == 0 ? s1 * d[n][2 + c] : fmaf(s1, d[n][2 + c], v[2]);
            zq[n][c] = ng == 0 ? b0 * qs[n][ng][c] : fmaf(b0, qs[n][ng][c], zq[n][c]);
            zq[n][2 + c] = ng == 0 ? b1 * qs[n][ng][c] : fmaf(b1, qs[n][ng][c], zq[n][2 + c]);
          }
      }
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[n][4 * r + i] = fmaf(s[n][4 * r + i], f[n][i & 1], zq[n][i]);
          if (!ALL && 16 * r + 8 * (i >> 1) + g >= valid) s[n][4 * r + i] = -INFINITY;
        }
    }
    float top[NH][2];
    bool grow = false;
    // The V scales, one token per lane. As bits they are ordered, and the zero
    // point below one does not change which power of two it reaches.
    const uint8_t* scales = rec + (lane >> 4) * 2 * KREC + KREC + KV4_CODES + 4 * (lane & 15);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      uint32_t x = *reinterpret_cast<const uint32_t*>(scales + 64 * i);
      if (!ALL && lane >= valid) x = 0;
      grow |= x >= KV4_R_SUM - __float_as_uint(rs[i]);
    }
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[n][c] = fmaxf(fmaxf(s[n][c], s[n][2 + c]), fmaxf(s[n][4 + c], s[n][6 + c]));
        grow |= top[n][c] > m[n][c] + KV4_LAZY;
      }
    if (__any_sync(0xffffffffu, grow)) {
      float move[NG];                        // of each group's sums
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        uint32_t x = *reinterpret_cast<const uint32_t*>(scales + 64 * i);
        if (!ALL && lane >= valid) x = 0;
        // a scale is below 2^11: what is not one (a NaN) moves r no further
        const int e = min(11, (int)(__reduce_max_sync(0xffffffffu, x) >> 23 & 255u) - 127);
        const float from = rs[i], to = fminf(from, __uint_as_float((uint32_t)(127 + KV4_R_TOP - max(e, KV4_R_MIN)) << 23));
        move[i] = __uint_as_float(__float_as_uint(to) - __float_as_uint(from) + (127u << 23));
        __syncwarp();
        if (lane == 0) rs[i] = to;
      }
      __syncwarp();
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = top[n][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          mx = fmaxf(mx, m[n][c]);
          const float corr = mx == -INFINITY ? 1.f : kv4_exp2(m[n][c] - mx);
          m[n][c] = mx;
          ref[n][c] = mx == -INFINITY ? 0.f : mx - KV4_P_BIAS;
          l[n][c] *= corr;
#pragma unroll
          for (int i = 0; i < NG; ++i) z[n][i][c] *= corr * move[i];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[n][i][c] *= corr * move[i * NG / 8];
            acc[n][i][2 + c] *= corr * move[i * NG / 8];
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[n][i] = kv4_exp2(s[n][i] - ref[n][i & 1]);
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) l[n][c] += (s[n][c] + s[n][2 + c]) + (s[n][4 + c] + s[n][6 + c]);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* vrec = rec + r * 2 * KREC + KREC;
      const uint4 v0 = *reinterpret_cast<const uint4*>(vrec + 16 * lane);
      const uint4 v1 = *reinterpret_cast<const uint4*>(vrec + 512 + 16 * lane);
      const uint32_t vw[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(vrec + KV4_CODES) + g;
#pragma unroll
      for (int ng = 0; ng < NG; ++ng) {
        uint32_t p0 = vp[ng * 16], p1 = vp[ng * 16 + 8];
        if (!ALL && 16 * r + g >= valid) p0 = 0;
        if (!ALL && 16 * r + g + 8 >= valid) p1 = 0;
        const float s0 = kv4_scale(p0) * rs[ng], s1 = kv4_scale(p1) * rs[ng];
        const float z0 = kv4_zero(p0), z1 = kv4_zero(p1);
        uint32_t w[NH][2];
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          const float* p = &s[n][4 * r];
          const __half2 h0 = __floats2half2_rn(p[0] * s0, p[1] * s0), h1 = __floats2half2_rn(p[2] * s1, p[3] * s1);
          w[n][0] = movm_t(*reinterpret_cast<const uint32_t*>(&h0));
          w[n][1] = movm_t(*reinterpret_cast<const uint32_t*>(&h1));
          z[n][ng][0] = fmaf(__low2float(h0), z0, fmaf(__low2float(h1), z1, z[n][ng][0]));
          z[n][ng][1] = fmaf(__high2float(h0), z0, fmaf(__high2float(h1), z1, z[n][ng][1]));
        }
#pragma unroll
        for (int j = 0; j < 8 / NG; ++j) {
          const int i = ng * (8 / NG) + j;
          const uint32_t x = vw[i], y = x >> 8;
#pragma unroll
          for (int n = 0; n < NH; ++n)
            mma_f16(acc[n][i], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, w[n][0], w[n][1]);
        }
      }
    }
  }

  // The result becomes NaN.
  __device__ __forceinline__ void poison() {
#pragma unroll
    for (int n = 0; n < NH; ++n) l[n][0] = l[n][1] = __uint_as_float(0x7fffffffu);
  }

  // Sum the lanes' shares and complete the output: afterwards acc[n][i][e] is
  // the unnormalised output of channel 16 i + g + 8 (e / 2), column
  // 8 n + 2 t + e % 2.
  __device__ __forceinline__ void finish() {
    float r[NG];                             // 2^r
#pragma unroll
    for (int i = 0; i < NG; ++i) r[i] = __uint_as_float((254u << 23) - __float_as_uint(rs[i]));
#pragma unroll
    for (int n = 0; n < NH; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
#pragma unroll
          for (int i = 0; i < NG; ++i) z[n][i][c] += __shfl_xor_sync(0xffffffffu, z[n][i][c], o);
        }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[n][i][e] = fmaf(acc[n][i][e], e < 2 ? 16777216.f : 1048576.f, z[n][i * NG / 8][e & 1]) * r[i * NG / 8];
    }
  }

  // A finished state as 9 NH rows of one float4 per lane: (m, m, l, l), then the
  // eight tiles, for each n.
  static constexpr int PART = 9 * NH * 32;   // float4s
  __device__ __forceinline__ void save(float4* part) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      __stcg(part + 9 * n * 32 + lane, make_float4(m[n][0], m[n][1], l[n][0], l[n][1]));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        __stcg(part + (9 * n + 1 + i) * 32 + lane, make_float4(acc[n][i][0], acc[n][i][1], acc[n][i][2], acc[n][i][3]));
    }
  }
  // Join up to eight saved states, in order. part(x): the x-th one.
  template <class Part>
  __device__ __forceinline__ void join(int count, Part part) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll 4
      for (int x = 0; x < count; ++x) {
        const float4 ml = __ldcg(part(x) + 9 * n * 32 + lane);
        m0 = fmaxf(m0, ml.x);
        m1 = fmaxf(m1, ml.y);
      }
      m[n][0] = m0;
      m[n][1] = m1;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
#pragma unroll 2
      for (int x = 0; x < count; ++x) {
        const float4* p = part(x) + 9 * n * 32 + lane;
        const float4 ml = __ldcg(p);
        float4 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __ldcg(p + 32 * (i + 1));
        // a part that saw no token counts nothing (a NaN sum goes on)
        const float e0 = ml.z == 0.f ? 0.f : kv4_exp2(ml.x - m0), e1 = ml.w == 0.f ? 0.f : kv4_exp2(ml.y - m1);
        l[n][0] += ml.z * e0;
        l[n][1] += ml.w * e1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[n][i][0] = fmaf(o[i].x, e0, acc[n][i][0]);
          acc[n][i][1] = fmaf(o[i].y, e1, acc[n][i][1]);
          acc[n][i][2] = fmaf(o[i].z, e0, acc[n][i][2]);
          acc[n][i][3] = fmaf(o[i].w, e1, acc[n][i][3]);
        }
      }
    }
  }

  // Normalise and store as bf16: column c's row is out + c * HD, `cols` columns
  // (VEC: rows are 4-byte aligned). A column that saw no token gives zeros.
  template <bool VEC>
  __device__ __forceinline__ void store(__nv_bfloat16* out, int cols) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const float i0 = l[n][0] != 0.f ? 1.f / l[n][0] : 0.f, i1 = l[n][1] != 0.f ? 1.f / l[n][1] : 0.f;
      // the transposed tile has column g's channels 2t, 2t + 1 side by side
      __nv_bfloat16* dst = out + (n * 8 + g) * HD + 2 * t;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = movm_t(pack_bf16(acc[n][i][2 * h] * i0, acc[n][i][2 * h + 1] * i1));
          if (n * 8 + g < cols) {
            if (VEC) {
              *reinterpret_cast<uint32_t*>(dst + 16 * i + 8 * h) = w;
            } else {
              reinterpret_cast<uint16_t*>(dst + 16 * i + 8 * h)[0] = (uint16_t)w;
              reinterpret_cast<uint16_t*>(dst + 16 * i + 8 * h)[1] = (uint16_t)(w >> 16);
            }
          }
        }
    }
  }
};

}  // namespace dsv
