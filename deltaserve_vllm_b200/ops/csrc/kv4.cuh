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
// 2^10.1, so that s * p (p a softmax weight below 2^5) and s * (c + z) fit fp16;
// the scale itself is bf16 so that small groups keep their relative precision.
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

__device__ __forceinline__ float kv4_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
// are undone by `f`. Output: O = sum p s c + sum p s z: p s is rounded to fp16
// (11 bits) for the matrix instruction, the second sum is one fp32 number per
// group and column.
constexpr float KV4_P_BIAS = 2.f;
constexpr float KV4_LAZY = 3.f;

template <int NG, int NH>
struct Kv4Warp {
  uint32_t q[NH][8][2];   // B fragments of the query, k-step by k-step
  float f[NH][2];         // score factor of columns 2t, 2t + 1
  float qs[NH][NG][2];    // scaled sum of the query over each group
  float acc[NH][8][4];    // sum p s c, channels 16 m + g (+ 8: times 16) x columns 2t, 2t + 1; times 2^-24
  float z[NH][NG][2];     // this lane's share of sum p s z
  float m[NH][2], l[NH][2];

  // `row(h)` gives the address of column h's 128 query values, null past the last one.
  template <class Row>
  __device__ __forceinline__ void begin(Row row, float scale_log2) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      float v[4][8];
      const __nv_bfloat16* src = row(n * 8 + g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (src != nullptr) w = *reinterpret_cast<const uint4*>(src + 32 * i + 8 * t);
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[i][2 * e] = __uint_as_float(x[e] << 16);
          v[i][2 * e + 1] = __uint_as_float(x[e] & 0xffff0000u);
        }
      }
      float amax = 0.f, sum[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) sum[i] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          amax = fmaxf(amax, fabsf(v[i][e]));
          sum[i * NG / 4] += v[i][e];
        }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
#pragma unroll
        for (int i = 0; i < NG; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      }
      // amax in [2^e, 2^(e+1)): scale by 2^(14 - e), e kept where that is a normal float
      const int e = min(127, max(-100, (int)((__float_as_uint(amax) >> 23) & 255u) - 127));
      const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
      const float down = up * 0.0625f;
      const float fh = scale_log2 * exp2f((float)(e + 10));   // 2^24 / up
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[n][2 * i][0] = pack_f16(v[i][0] * up, v[i][4] * up);
        q[n][2 * i][1] = pack_f16(v[i][1] * down, v[i][5] * down);
        q[n][2 * i + 1][0] = pack_f16(v[i][2] * up, v[i][6] * up);
        q[n][2 * i + 1][1] = pack_f16(v[i][3] * down, v[i][7] * down);
      }
      // the scores' columns are 2t, 2t + 1: fetch those columns' factors
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 4 * (2 * t + c);
        f[n][c] = __shfl_sync(0xffffffffu, fh, from);
#pragma unroll
        for (int i = 0; i < NG; ++i) qs[n][i][c] = scale_log2 * __shfl_sync(0xffffffffu, sum[i], from);
        m[n][c] = -INFINITY;
        l[n][c] = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) z[n][i][c] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
    }
  }

  // One K and V record (`rec` points at K's; 16-byte aligned, shared or global
  // memory). `seen(token, column)` says whether a column sees token 0..15.
  template <class Seen>
  __device__ __forceinline__ void tile(const uint8_t* rec, Seen seen) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint8_t* vrec = rec + kv4_record(NG);
    const uint4 k0 = *reinterpret_cast<const uint4*>(rec + g * 64 + t * 16);
    const uint4 k1 = *reinterpret_cast<const uint4*>(rec + 512 + g * 64 + t * 16);
    const uint32_t kw0[4] = {k0.x, k0.y, k0.z, k0.w}, kw1[4] = {k1.x, k1.y, k1.z, k1.w};
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(rec + KV4_CODES);
    const uint32_t* vp = reinterpret_cast<const uint32_t*>(vrec + KV4_CODES);
    float s[NH][4];
#pragma unroll
    for (int n = 0; n < NH; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
    float zq[NH][4];
#pragma unroll
    for (int n = 0; n < NH; ++n) zq[n][0] = zq[n][1] = zq[n][2] = zq[n][3] = 0.f;
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
      const uint32_t p0 = kp[ng * 16 + g], p1 = kp[ng * 16 + 8 + g];
      const float s0 = kv4_scale(p0), s1 = kv4_scale(p1);
      const float b0 = s0 * kv4_zero(p0), b1 = s1 * kv4_zero(p1);
#pragma unroll
      for (int n = 0; n < NH; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          s[n][c] = fmaf(s0, d[n][c], s[n][c]);
          s[n][2 + c] = fmaf(s1, d[n][2 + c], s[n][2 + c]);
          zq[n][c] = fmaf(b0, qs[n][ng][c], zq[n][c]);
          zq[n][2 + c] = fmaf(b1, qs[n][ng][c], zq[n][2 + c]);
        }
      }
    }
    bool grow = false;
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = n * 8 + 2 * t + c;
        s[n][c] = seen(g, col) ? fmaf(s[n][c], f[n][c], zq[n][c]) : -INFINITY;
        s[n][2 + c] = seen(g + 8, col) ? fmaf(s[n][2 + c], f[n][c], zq[n][2 + c]) : -INFINITY;
        grow |= fmaxf(s[n][c], s[n][2 + c]) > m[n][c] + KV4_LAZY;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(s[n][c], s[n][2 + c]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          mx = fmaxf(mx, m[n][c]);
          const float corr = mx == -INFINITY ? 1.f : kv4_exp2(m[n][c] - mx);
          m[n][c] = mx;
          l[n][c] *= corr;
#pragma unroll
          for (int i = 0; i < NG; ++i) z[n][i][c] *= corr;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[n][i][c] *= corr;
            acc[n][i][2 + c] *= corr;
          }
        }
    }
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float ref = m[n][c] == -INFINITY ? 0.f : m[n][c] - KV4_P_BIAS;
        s[n][c] = kv4_exp2(s[n][c] - ref);
        s[n][2 + c] = kv4_exp2(s[n][2 + c] - ref);
        l[n][c] += s[n][c] + s[n][2 + c];
      }
#pragma unroll
    for (int ng = 0; ng < NG; ++ng) {
      const uint32_t p0 = vp[ng * 16 + g], p1 = vp[ng * 16 + 8 + g];
      const float s0 = kv4_scale(p0), s1 = kv4_scale(p1);
      const float b0 = s0 * kv4_zero(p0), b1 = s1 * kv4_zero(p1);
      uint32_t w[NH][2];
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        // an unseen token's weight is 0 whatever its record holds
        float u[4];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const bool on0 = s[n][c] != 0.f, on1 = s[n][2 + c] != 0.f;
          u[c] = on0 ? s[n][c] * s0 : 0.f;
          u[2 + c] = on1 ? s[n][2 + c] * s1 : 0.f;
          z[n][ng][c] += (on0 ? s[n][c] * b0 : 0.f) + (on1 ? s[n][2 + c] * b1 : 0.f);
        }
        w[n][0] = movm_t(pack_f16(u[0], u[1]));
        w[n][1] = movm_t(pack_f16(u[2], u[3]));
      }
#pragma unroll
      for (int j = 0; j < 8 / NG; ++j) {
        const int i = ng * (8 / NG) + j;
        const uint32_t x = *reinterpret_cast<const uint32_t*>(vrec + 512 * (i / 4) + 16 * lane + 4 * (i % 4));
        const uint32_t y = x >> 8;
#pragma unroll
        for (int n = 0; n < NH; ++n)
          mma_f16(acc[n][i], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, w[n][0], w[n][1]);
      }
    }
  }

  // Sum the lanes' shares; afterwards `out(n, i, e)` is the unnormalised output
  // of channel 16 i + g + 8 (e / 2), column 8 n + 2 t + e % 2.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
#pragma unroll
          for (int i = 0; i < NG; ++i) z[n][i][c] += __shfl_xor_sync(0xffffffffu, z[n][i][c], o);
        }
  }
  __device__ __forceinline__ float out(int n, int i, int e) const {
    return fmaf(acc[n][i][e], e < 2 ? 16777216.f : 1048576.f, z[n][i * NG / 8][e & 1]);
  }
};

}  // namespace dsv
