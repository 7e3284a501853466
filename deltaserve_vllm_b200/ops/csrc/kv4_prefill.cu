// Causal attention of new tokens over the 4-bit paged KV cache on the
// 5th-generation tensor cores (format: kv4.cuh): packed sequences of any
// lengths, each with its cached context, grouped query heads.
//
// The reference project prefills over its serving library's bf16 pages; this is
// the same function over the values the codes stand for.
//
// One CTA = one KV head and up to 256 query rows of one sequence as two 128-row
// tiles; a row is (query, head of the group), queries first, so one K / V tile
// serves every head of the group and the causal triangle wastes 128 / group
// queries per tile only. 512 threads in four roles:
//
//   warps 0-3, 4-7   softmax of tile 0 and tile 1, one row per thread: scores
//                    from TMEM, mask, running maximum, P as fp16 back into the
//                    scores' TMEM columns, lazy rescaling of O.
//   warps 8-11       dequantise: 128 keys at a time from global memory through
//                    registers (prefetched one tile ahead) into swizzled shared
//                    memory, K then V, two stages each.
//   warp 12          issues the MMAs: S_x = Q_x K^T, then O_x += P_x V with P
//                    from TMEM. Tile 0's softmax runs while tile 1's products do.
//
// Operands are fp16 (fp32 accumulators): a value s (c + z) of the 4-bit format is
// off by at most 2^-10 of itself (two roundings to 11 bits, see p4_values), where
// bf16 operands would double the result's own rounding error. fp16 has few
// exponents, so every operand enters relative to a power of two of its own: K to
// that of the largest scale of a warp's 32 keys (undone on the score), V to that of
// the largest scale so far of each group of channels (a larger one rescales O, as a
// larger maximum does), each query row to that of its largest magnitude, and P to a
// reference that puts the largest weight between 2^9 and 2^15. A value keeps its
// bits down to 2^-24 of the largest, a weight to 2^-23. (With fixed divisors of 16
// values near 1e-5 were off by 3 %, and weights of 2^-16 beside a dominant key by
// their rounding to subnormals.)
//
// K is stored as [keys x channels], V as [channels x keys] (both K-major for
// their product): the code pairs that one mask yields, channels (c, c + 4) of
// K and tokens (2t, 2t + 1) of V, are then neighbours in shared memory. For K
// the order of the eight channels of a 16-byte unit is that of the pairs
// (0, 4, 1, 5, 2, 6, 3, 7), and Q is stored in the same order.
//
// Shared memory: Q 64 KB, K 2 x 32 KB, V 2 x 32 KB, units and factors. TMEM: S0, S1, O0, O1 of 128
// columns each; P_x takes the first 64 columns of S_x.
//
// Measured (32 / 8 heads, groups of 64): 2048 tokens after 29952 in 1250 us,
// 833 TFLOP/s. Its 256 CTAs are two rounds of 148 (86 % of the SMs' time); in a
// CTA the products (2048 cycles per 128 keys at full rate), the exponentials (2048
// at 16 a cycle) and the operands' shared-memory traffic (about 2048) overlap only
// in part (tensor pipe 56 % busy, exponentials 44 %), and with the conversions
// taken out an earlier step at 709 ran at 955.
//
// Every wait is bounded (common.cuh).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "attn_tc.cuh"
#include "kv4.cuh"

int dsv_kv4_groups(const torch::Tensor& cache, const char* op);
int64_t dsv_kv4_workspace_bytes();

namespace dsv {

constexpr int P4_THREADS = 512;
constexpr int P4_CHUNK = 128 * 128;          // [128 rows x 64 columns] fp16, bytes
constexpr int P4_TILE = 2 * P4_CHUNK;
constexpr int P4_SMEM = 6 * P4_TILE + 1024 + 256 * 4 + 256 + 256;
constexpr float P4_P_BIAS = 9.f;
constexpr float P4_LAZY = 6.f;                // 4: 12 packed sequences 271 us in place of 261, 8 and a bias of 7: 259
constexpr int P4_PART = HD + 4;              // floats of a row's partial result
constexpr uint32_t P4_IDESC = (1u << 4) | (128u >> 3) << 17 | (128u >> 4) << 24;   // f16 x f16 -> f32, 128 x 128

enum : int {
  kErrP4K = 0x4401,
  kErrP4V = 0x4402,
  kErrP4S = 0x4403,
  kErrP4P = 0x4404,
  kErrP4O = 0x4405,
  kErrP4KEmpty = 0x4406,
  kErrP4VEmpty = 0x4407,
  kErrP4Top = 0x4408,
};

struct Prefill4Args {
  const __nv_bfloat16* q;   // [T, Hq * 128], row stride q_stride
  int64_t q_stride;
  const uint8_t* cache;
  const int* tables;        // [S, max_pages]
  const int* cu_q;          // [S + 1]
  const int* ctx;           // [S]
  __nv_bfloat16* out;
  int64_t out_stride;
  int seqs, rows, max_pages, num_pages, kv_heads, group, sub;
  int tile_rows;            // query rows per CTA: 128 or 256
  int splits;               // CTAs that share a tile's keys (128-row tiles only)
  float* part;              // [grid x, Hkv, splits, 128 rows, P4_PART]: unnormalised output, maximum, sum
  float scale_log2;
};

// D[tmem] (+)= A[tmem] * B[smem]^T, 16-bit operands.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 lanes x 16 columns (common.cuh has the 32-column forms): the softmax warps
// have no 32 registers to spare beside a row of scores.
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

template <int N>
__device__ __forceinline__ void reg_grow() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_shrink() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

struct P4Tile {
  int seq, local;           // sequence (-1: past the last tile) and which of its query tiles
};
// The `left`-th tile of the packed sequences: a sequence's last, longest tile first.
// A sequence whose rows are not rows of q has none, and is an error.
__device__ __forceinline__ P4Tile p4_tile(const Prefill4Args& a, int left) {
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < a.seqs; s0 += 32) {
    int n = 0;
    if (s0 + lane < a.seqs) {
      const int begin = a.cu_q[s0 + lane], end = a.cu_q[s0 + lane + 1];
      if (begin < 0 || end < begin || end > a.rows) set_error(kErrShape);
      else n = ((end - begin) * a.group + a.tile_rows - 1) / a.tile_rows;
    }
    int up = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, up > left);
    if (past != 0) {
      const int at = __ffs(past) - 1;
      return {s0 + at, __shfl_sync(0xffffffffu, up, at) - 1 - left};
    }
    left -= __shfl_sync(0xffffffffu, up, 31);
  }
  return {-1, 0};
}

// The values s (c + z) of a word's eight codes as four pairs (code i, code i + 4),
// relative to 2^(e - 5), where 2^e is the power of two of the largest scale: the
// masked codes are the fp16 subnormals c 2^-24 (c 2^-20), `z` is the zero point
// times 2^-9 and `s` the scale times 2^(14 - e). Two roundings: c + z is exact where
// the zero point's unit is no finer than the sum's, else off by up to 2^-11 of
// itself, and the product by as much again. Rounding s z once for a whole group
// instead cost as many instructions and, being the same error for all its channels,
// moved the scores of long contexts by up to a bf16 step of the output.
__device__ __forceinline__ void p4_values(uint32_t w, __half2 s, __half2 z, uint32_t (&v)[4]) {
  const __half2 up0 = __float2half2_rn(32768.f), up1 = __float2half2_rn(2048.f);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t m0 = w & 0x000f000fu, m1 = w & 0x00f000f0u;
    const __half2 v0 = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&m0), up0, z), s);
    const __half2 v1 = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&m1), up1, z), s);
    v[2 * i] = *reinterpret_cast<const uint32_t*>(&v0);
    v[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&v1);
    w >>= 8;
  }
}
// A (scale, zero point) word as those two factors: fp16 s 2^(14 - e) in the low half, z 2^-9 in the high half.
__device__ __forceinline__ uint32_t p4_factors(uint32_t word, int e) {
  return pack_f16(kv4_scale(word) * __uint_as_float((uint32_t)(127 + 14 - e) << 23), kv4_zero(word) * 0.001953125f);
}
// The exponent of a word's scale, kept where 2^(14 - e) is finite. Scales are
// below 2^11; what is not one (a NaN) counts as the largest.
constexpr int P4_E_MIN = -110;
__device__ __forceinline__ int p4_exponent(uint32_t word) {
  return min(11, max(P4_E_MIN, (int)(word >> 23 & 255u) - 127));
}
// 2^(e - 5): what a stored 1 stands for.
__device__ __forceinline__ float p4_unit(int e) { return __uint_as_float((uint32_t)(127 - 5 + e) << 23); }

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
        "l"(reinterpret_cast<unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d))
      : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int NG>
__global__ void __launch_bounds__(P4_THREADS, 1) prefill4_kernel(const Prefill4Args a) {
  extern __shared__ uint8_t p4_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p4_smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                       // [2][tile]
  uint8_t* sK = sQ + 2 * P4_TILE;           // [2][tile]
  uint8_t* sV = sK + 2 * P4_TILE;           // [2][tile]
  float* sF = reinterpret_cast<float*>(sV + 2 * P4_TILE);   // [256] score factor of each row
  uint64_t* bars = reinterpret_cast<uint64_t*>(sF + 256);
  uint64_t* k_full = bars + 0;    // [2]
  uint64_t* v_full = bars + 2;    // [2]
  uint64_t* k_empty = bars + 4;   // [2]
  uint64_t* v_empty = bars + 6;   // [2]
  uint64_t* s_full = bars + 8;    // [2] by tile
  uint64_t* p_full = bars + 10;   // [2] by tile
  uint64_t* o_done = bars + 12;   // [2] by tile
  uint64_t* drain = bars + 14;
  uint64_t* top_full = bars + 15;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  // Units of the operands, by key tile modulo 4: a slot is written again when the
  // scores of two tiles later have been taken, by when every softmax has read it.
  float* k_unit = reinterpret_cast<float*>(bars + 32);   // [4][dequantising warp]
  float* v_unit = k_unit + 16;                           // [4][group]
  uint32_t* v_top = reinterpret_cast<uint32_t*>(v_unit + 16);   // [2][group][warp] largest words of a tile

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kvh = blockIdx.y;

  const P4Tile tile = p4_tile(a, blockIdx.x);
  const int seq = tile.seq, local = tile.local;
  if (seq < 0) return;
  const int q_begin = a.cu_q[seq], q_len = a.cu_q[seq + 1] - q_begin;
  const int ctx = min(a.ctx[seq], a.max_pages * a.sub * 16);
  const int pos0 = ctx - q_len;                           // position of the first new token
  const int row0 = local * a.tile_rows;
  const int rows = min(a.tile_rows, q_len * a.group - row0);
  const int* tab = a.tables + (size_t)seq * a.max_pages;
  // keys that the last query of tile x sees, and how many key tiles that is
  int n_kb[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int last = min(rows, (x + 1) * 128) - 1;
    n_kb[x] = last >= x * 128 ? max(0, pos0 + (row0 + last) / a.group + 1 + 127) / 128 : 0;
  }
  // this split's key tiles: kb0 onwards
  int kb0 = 0;
  if (a.splits > 1) {
    const int per = max(2, (n_kb[0] + a.splits - 1) / a.splits);
    kb0 = (int)blockIdx.z * per;
    n_kb[0] = max(0, min(per, n_kb[0] - kb0));
  }
  const int n_max = max(n_kb[0], n_kb[1]);
  const int kv_end = pos0 + (row0 + rows - 1) / a.group + 1;

  if (threadIdx.x == 0) {
    if (a.ctx[seq] > ctx) set_error(kErrShape);           // longer than its table: only those pages are seen
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 128);
      mbar_init(&v_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    mbar_init(top_full, 4);
    fence_barrier_init();
  }
  if (warp == 12) tmem_alloc(tmem_slot, 512);
  // Q: two threads per row, 64 channels each.
  {
    const int r = threadIdx.x / 2, half = threadIdx.x & 1;
    const bool ok = r < rows;
    const int rr = row0 + (ok ? r : 0);
    const __nv_bfloat16* src = a.q + (int64_t)(q_begin + rr / a.group) * a.q_stride +
                               (int64_t)(kvh * a.group + rr % a.group) * HD + half * 64;
    uint4 v[8];
    float amax = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      v[u] = ok ? *reinterpret_cast<const uint4*>(src + u * 8) : make_uint4(0, 0, 0, 0);
      const uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(x[e] << 16)), fabsf(__uint_as_float(x[e] & 0xffff0000u))));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    const int e = min(126, max(-100, (int)((__float_as_uint(amax) >> 23) & 255u) - 127));
    const float up = __uint_as_float((uint32_t)(127 - e) << 23);
    if (half == 0) sF[r] = a.scale_log2 * exp2f((float)e);
    uint8_t* dst = sQ + (r >> 7) * P4_TILE + half * P4_CHUNK + (r & 127) * 128;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(x[i] << 16) * up;
        f[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u) * up;
      }
      *reinterpret_cast<uint4*>(dst + ((u ^ (r & 7)) << 4)) =
          make_uint4(pack_f16(f[0], f[4]), pack_f16(f[1], f[5]), pack_f16(f[2], f[6]), pack_f16(f[3], f[7]));
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    // -------------------------------------------------------------- softmax
    reg_grow<192>();
    const int x = warp >> 2;
    const int r = (warp & 3) * 32 + lane;
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_lane + x * 128, t_o = t_lane + 256 + x * 128;
    const int row = row0 + x * 128 + r;                     // row of the sequence
    const bool row_ok = x * 128 + r < rows;
    const int seen = pos0 + row / a.group + 1;              // keys that this row sees
    const float f = sF[x * 128 + r];
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const int n = n_kb[x];
    for (int j = 0; j < n; ++j) {
      if (!__all_sync(0xffffffffu, kv4_wait(&s_full[x], (uint32_t)j & 1u, kErrP4S))) { ok = false; break; }
      tc_fence_after();
      float s[128];
      {
        uint32_t v0[32], v1[32], v2[32], v3[32];
        tmem_ld_32x32b_x32(t_s + 0, v0);
        tmem_ld_32x32b_x32(t_s + 32, v1);
        tmem_ld_32x32b_x32(t_s + 64, v2);
        tmem_ld_32x32b_x32(t_s + 96, v3);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s[i] = __uint_as_float(v0[i]);
          s[32 + i] = __uint_as_float(v1[i]);
          s[64 + i] = __uint_as_float(v2[i]);
          s[96 + i] = __uint_as_float(v3[i]);
        }
      }
      const int lim = seen - (kb0 + j) * 128;
      if (__any_sync(0xffffffffu, lim < 128)) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= lim) s[i] = -INFINITY;
      }
      float red[4], fc[4];
      {
        const float4 u = *reinterpret_cast<const float4*>(k_unit + (j & 3) * 4);
        const float uc[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) fc[c] = fminf(fmaxf(f * uc[c], 1.2e-38f), 3e38f);   // 0 would make a masked key NaN
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) red[c] = fmaxf(s[32 * c], s[32 * c + 1]);
#pragma unroll
      for (int i = 2; i < 32; i += 2)
#pragma unroll
        for (int c = 0; c < 4; ++c) red[c] = max3(red[c], s[32 * c + i], s[32 * c + i + 1]);
      const float row_max = fmaxf(fmaxf(fc[0] * red[0], fc[1] * red[1]), fmaxf(fc[2] * red[2], fc[3] * red[3]));
      // The reference maximum moves only when it is exceeded by 2^6: P stays
      // below 2^15 in fp16 and the common factor cancels in O / l.
      const bool move = m == -INFINITY || row_max > m + P4_LAZY;
      const float mx = move ? fmaxf(m, row_max) : m;
      const float corr = m == -INFINITY ? 0.f : (move ? kv4_exp2(m - mx) : 1.f);
      const float ref = mx == -INFINITY ? 0.f : mx - P4_P_BIAS;
      l *= corr;
      m = mx;
      // s_full of this tile was committed after the last product into O
      bool scale_o = corr != 1.f;
      const uint32_t* unit_now = reinterpret_cast<const uint32_t*>(v_unit) + (j & 3) * 4;
      const uint32_t* unit_before = reinterpret_cast<const uint32_t*>(v_unit) + (j - 1 & 3) * 4;
#pragma unroll
      for (int i = 0; i < NG; ++i) scale_o |= unit_now[i] != unit_before[i];
      if (j > 0 && __any_sync(0xffffffffu, scale_o)) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int i = c * NG / 8;
          const float by = corr * __uint_as_float(unit_before[i] - unit_now[i] + (127u << 23));
          uint32_t v[16];
          tmem_ld_x16(t_o + c * 16, v);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * by);
          tmem_st_x16(t_o + c * 16, v);
        }
      }
      const float2 r2 = make_float2(-ref, -ref);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t p[16];
        const float2 f2 = make_float2(fc[c], fc[c]);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float2 e = fma2(make_float2(s[c * 32 + 2 * i], s[c * 32 + 2 * i + 1]), f2, r2);
          e = make_float2(kv4_exp2(e.x), kv4_exp2(e.y));
          sum[i & 1] = add2(sum[i & 1], e);
          p[i] = pack_f16(e.x, e.y);
        }
        tmem_st_x16(t_s + c * 16, p);
      }
      sum[0] = add2(sum[0], sum[1]);
      l += sum[0].x + sum[0].y;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, kv4_wait(&o_done[x], 0, kErrP4O));
    const float* unit = v_unit + (n - 1 & 3) * 4;           // of O
    if (ok && a.splits > 1) {
      tc_fence_after();
      float* dst = a.part + ((((size_t)blockIdx.x * a.kv_heads + kvh) * a.splits + blockIdx.z) * 128 + r) * P4_PART;
      if (x == 0) {
        *reinterpret_cast<float2*>(dst + HD) = make_float2(m, l);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (n == 0) break;
          uint32_t v[16];
          tmem_ld_x16(t_o + c * 16, v);
          tmem_ld_wait();
          const float by = unit[c * NG / 8];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<float4*>(dst + c * 16 + u * 4) =
                make_float4(__uint_as_float(v[4 * u]) * by, __uint_as_float(v[4 * u + 1]) * by,
                            __uint_as_float(v[4 * u + 2]) * by, __uint_as_float(v[4 * u + 3]) * by);
        }
      }
    } else if (ok) {
      tc_fence_after();
      const float inv = l != 0.f ? 1.f / l : 0.f;           // a row that sees no key gives zeros
      __nv_bfloat16* dst = a.out + (int64_t)(q_begin + row / a.group) * a.out_stride +
                           (int64_t)(kvh * a.group + row % a.group) * HD;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        float by = 0.f;
        if (n > 0) {
          tmem_ld_32x32b_x32(t_o + c * 32, v);
          tmem_ld_wait();
          by = unit[c * NG / 4];
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0;
        }
        if (row_ok) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack2_bf16(__uint_as_float(v[u * 8 + 2 * e]) * inv * by,
                                __uint_as_float(v[u * 8 + 2 * e + 1]) * inv * by);
            *reinterpret_cast<uint4*>(dst + c * 32 + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  } else if (warp < 12) {
    // -------------------------------------------------------------- dequantise
    reg_shrink<88>();
    const int w4 = warp - 8;
    // The warp's 32 keys of a tile are two records; lane l has token l % 16 of
    // record l / 16: its K row, and its K and V scales and zero points.
    const int key = w4 * 32 + lane;
    const int g = lane >> 2, t = lane & 3;
    uint4 kc[4], vc[2][2];
    uint32_t kp[NG], vp[NG];
    // The record's place, moved by a tile (8 records) at a time, and its page a tile ahead of its use.
    const int step_page = 8 / a.sub, step_off = 8 % a.sub;
    int at_key = kb0 * 128 + key;
    int at_page = (at_key / 16) / a.sub, at_off = (at_key / 16) % a.sub;
    int page = 0;
    const uint8_t* rec = nullptr;               // of the tile to load; null past the end
    bool in = false;                            // its token exists
    auto next = [&]() {                         // the looked-up record's address, then the next look-up
      rec = nullptr;
      in = at_key < kv_end;
      if (at_key - (lane & 15) < kv_end) {
        if ((unsigned)page >= (unsigned)a.num_pages) {              // read another page instead, and say so
          set_error(kErrShape);
          page = 0;
        }
        rec = a.cache + (((size_t)page * a.kv_heads + kvh) * a.sub + at_off) * (2 * kv4_record(NG));
      }
      at_key += 128;
      at_page += step_page;
      at_off += step_off;
      if (at_off >= a.sub) {
        at_off -= a.sub;
        ++at_page;
      }
      if (at_key - (lane & 15) < kv_end) page = tab[at_page];
    };
    auto load_k = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        kc[i] = in ? *reinterpret_cast<const uint4*>(rec + (lane & 15) * 64 + i * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NG; ++i)
        kp[i] = in ? *reinterpret_cast<const uint32_t*>(rec + KV4_CODES + 64 * i + 4 * (lane & 15)) : 0u;
      // a key that no query sees is a zero row whatever its record holds
#pragma unroll
      for (int i = 0; i < NG; ++i)
        vp[i] = in ? *reinterpret_cast<const uint32_t*>(rec + kv4_record(NG) + KV4_CODES + 64 * i + 4 * (lane & 15)) : 0u;
    };
    auto load_v = [&]() {
      const uint8_t* v = rec != nullptr ? rec + kv4_record(NG) : nullptr;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(
            __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(v), 16 * b));
#pragma unroll
        for (int i = 0; i < 2; ++i)
          vc[b][i] = p != nullptr ? *reinterpret_cast<const uint4*>(p + i * 512 + lane * 16) : make_uint4(0, 0, 0, 0);
      }
    };
    int ev[NG];                                 // V's exponents, the largest scale so far
#pragma unroll
    for (int i = 0; i < NG; ++i) ev[i] = P4_E_MIN;
    if (n_max > 0) {
      if (at_key - (lane & 15) < kv_end) page = tab[at_page];
      next();
      load_k();
      load_v();
    }
    for (int j = 0; j < n_max; ++j) {
      const int st = j & 1;
      const uint32_t ph = ((uint32_t)(j >> 1) & 1u) ^ 1u;
      if (!__all_sync(0xffffffffu, kv4_wait(&k_empty[st], ph, kErrP4KEmpty))) break;
      // The tile's units. The warps exchange V's largest words through a barrier
      // whose wait is bounded: one that gave up does not hold the others.
      uint32_t top = kp[0];
#pragma unroll
      for (int i = 1; i < NG; ++i) top = max(top, kp[i]);
      const int ek = p4_exponent(__reduce_max_sync(0xffffffffu, top));
      uint32_t* tops = v_top + (j & 1) * 16;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const uint32_t x = __reduce_max_sync(0xffffffffu, vp[i]);
        if (lane == 0) tops[4 * i + w4] = x;
      }
      if (lane == 0) {
        k_unit[(j & 3) * 4 + w4] = p4_unit(ek);
        mbar_arrive(top_full);
      }
      if (!__all_sync(0xffffffffu, kv4_wait(top_full, (uint32_t)j & 1u, kErrP4Top))) break;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(tops + 4 * i);
        ev[i] = max(ev[i], p4_exponent(max(max(x.x, x.y), max(x.z, x.w))));
        if (w4 == 0 && lane == 0) v_unit[(j & 3) * 4 + i] = p4_unit(ev[i]);
      }
      {
        uint8_t* dst = sK + st * P4_TILE + key * 128;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          const uint32_t f = p4_factors(kp[i], ek);
          const uint32_t f0 = __byte_perm(f, f, 0x1010), f1 = __byte_perm(f, f, 0x3232);
          const __half2 sc = *reinterpret_cast<const __half2*>(&f0), sz = *reinterpret_cast<const __half2*>(&f1);
#pragma unroll
          for (int e = i * (4 / NG); e < (i + 1) * (4 / NG); ++e)   // word e of 16 bytes h: channels 32 e + 8 h
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const uint32_t w = e == 0 ? kc[h].x : e == 1 ? kc[h].y : e == 2 ? kc[h].z : kc[h].w;
              uint32_t v[4];
              p4_values(w, sc, sz, v);
              const int u = 4 * e + h;                      // 16-byte unit of the row
              *reinterpret_cast<uint4*>(dst + (u >> 3) * P4_CHUNK + (((u & 7) ^ (key & 7)) << 4)) =
                  make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&k_full[st]);
      uint32_t ss[NG];                                      // the factors of this lane's token
#pragma unroll
      for (int i = 0; i < NG; ++i) ss[i] = p4_factors(vp[i], ev[i]);
      if (j + 1 < n_max) {
        next();
        load_k();
      }
      if (!__all_sync(0xffffffffu, kv4_wait(&v_empty[st], ph, kErrP4VEmpty))) break;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int r = w4 * 2 + b;                           // record of the tile
        uint8_t* dst = sV + st * P4_TILE + (r >> 2) * P4_CHUNK + g * 128 + 4 * t;
        const int u = 2 * (r & 3);                          // 16-byte unit (8 tokens) of the row; u + 1 the late half
        uint8_t* d0 = dst + ((u ^ g) << 4);
        uint8_t* d1 = dst + (((u + 1) ^ g) << 4);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          // scales and zero points of tokens 2t, 2t + 1 and 2t + 8, 2t + 9
          uint32_t sc[2], sz[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = __shfl_sync(0xffffffffu, ss[i], 16 * b + 8 * h + 2 * t);
            const uint32_t y = __shfl_sync(0xffffffffu, ss[i], 16 * b + 8 * h + 2 * t + 1);
            sc[h] = __byte_perm(x, y, 0x5410);
            sz[h] = __byte_perm(x, y, 0x7632);
          }
#pragma unroll
          for (int q = 0; q < 8 / NG; ++q) {
            const int mt = i * (8 / NG) + q;                // channels 16 mt + g and + 8
            const uint4& c = vc[b][mt / 4];
            const uint32_t w = mt % 4 == 0 ? c.x : mt % 4 == 1 ? c.y : mt % 4 == 2 ? c.z : c.w;
            uint32_t v[4], late[4];
            p4_values(w, *reinterpret_cast<const __half2*>(&sc[0]), *reinterpret_cast<const __half2*>(&sz[0]), v);
            p4_values(w, *reinterpret_cast<const __half2*>(&sc[1]), *reinterpret_cast<const __half2*>(&sz[1]), late);
            *reinterpret_cast<uint32_t*>(d0 + mt * 2048) = v[0];
            *reinterpret_cast<uint32_t*>(d0 + mt * 2048 + 1024) = v[1];
            *reinterpret_cast<uint32_t*>(d1 + mt * 2048) = late[2];
            *reinterpret_cast<uint32_t*>(d1 + mt * 2048 + 1024) = late[3];
          }
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&v_full[st]);
      if (j + 1 < n_max) load_v();
    }
  } else {
    reg_shrink<40>();
    if (warp == 12 && lane == 0 && n_max > 0) {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t q_addr = smem_u32(sQ), k_addr = smem_u32(sK), v_addr = smem_u32(sV);
      auto scores = [&](int x, int j) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          tc_mma_f16(tmem + x * 128, desc_kmajor(q_addr + x * P4_TILE, kk, P4_CHUNK),
                     desc_kmajor(k_addr + (j & 1) * P4_TILE, kk, P4_CHUNK), P4_IDESC, kk > 0 ? 1u : 0u);
        tc_commit(&s_full[x]);
      };
      auto output = [&](int x, int j) -> bool {
        if (!kv4_wait(&p_full[x], (uint32_t)j & 1u, kErrP4P)) return false;
        if (!kv4_wait(&v_full[j & 1], (uint32_t)(j >> 1) & 1u, kErrP4V)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)
          tc_mma_f16_ts(tmem + 256 + x * 128, tmem + x * 128 + kk * 8,
                        desc_kmajor(v_addr + (j & 1) * P4_TILE, kk, P4_CHUNK), P4_IDESC, (j > 0 || kk > 0) ? 1u : 0u);
        if (j == n_kb[x] - 1) tc_commit(&o_done[x]);
        return true;
      };
      bool ok = kv4_wait(&k_full[0], 0, kErrP4K);
      if (ok) {
        tc_fence_after();
        if (n_kb[0] > 0) scores(0, 0);
        if (n_kb[1] > 0) scores(1, 0);
        tc_commit(&k_empty[0]);
      }
      for (int j = 0; j < n_max && ok; ++j) {
        if (j < n_kb[0] && !output(0, j)) break;
        const bool more = j + 1 < n_max;
        if (more) {
          if (!kv4_wait(&k_full[(j + 1) & 1], (uint32_t)((j + 1) >> 1) & 1u, kErrP4K)) break;
          tc_fence_after();
          if (j + 1 < n_kb[0]) scores(0, j + 1);
        }
        if (j < n_kb[1] && !output(1, j)) break;
        tc_commit(&v_empty[j & 1]);
        if (more) {
          if (j + 1 < n_kb[1]) scores(1, j + 1);
          tc_commit(&k_empty[(j + 1) & 1]);
        }
      }
      // Every product has finished before the CTA gives its memory back.
      tc_commit(drain);
      kv4_drain(drain, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the splits of a tile: one warp per row, four channels per lane.
// grid (tile, KV head, 16), 8 rows per CTA.
__global__ void __launch_bounds__(256) prefill4_join_kernel(const Prefill4Args a) {
  const P4Tile tile = p4_tile(a, blockIdx.x);
  if (tile.seq < 0) return;
  const int lane = threadIdx.x & 31, kvh = blockIdx.y;
  const int r = blockIdx.z * 8 + threadIdx.x / 32;
  const int q_begin = a.cu_q[tile.seq], q_len = a.cu_q[tile.seq + 1] - q_begin;
  const int row = tile.local * 128 + r;
  if (row >= q_len * a.group) return;
  const float* part = a.part + ((((size_t)blockIdx.x * a.kv_heads + kvh) * a.splits) * 128 + r) * P4_PART;
  const size_t step = (size_t)128 * P4_PART;
  float M = -INFINITY, L = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, part[s * step + HD]);
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(part + s * step + HD);
    const float4 v = *reinterpret_cast<const float4*>(part + s * step + 4 * lane);
    if (ml.y == 0.f) continue;               // saw no key (a NaN sum goes on)
    const float e = kv4_exp2(ml.x - M);
    L += ml.y * e;
    o.x = fmaf(v.x, e, o.x);
    o.y = fmaf(v.y, e, o.y);
    o.z = fmaf(v.z, e, o.z);
    o.w = fmaf(v.w, e, o.w);
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  __nv_bfloat16* dst = a.out + (int64_t)(q_begin + row / a.group) * a.out_stride +
                       (int64_t)(kvh * a.group + row % a.group) * HD + 4 * lane;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
}

template <int NG>
static void prefill4_launch(const Prefill4Args& a, dim3 grid, cudaStream_t stream) {
  static const cudaError_t attr =
      cudaFuncSetAttribute(prefill4_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, P4_SMEM);
  C10_CUDA_CHECK(attr);
  prefill4_kernel<NG><<<grid, P4_THREADS, P4_SMEM, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (a.splits > 1) {
    prefill4_join_kernel<<<dim3(grid.x, grid.y, 16), 256, 0, stream>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

}  // namespace dsv

// ---------------------------------------------------------------- bindings

// Returns the number of kernels launched.
int64_t dsv_paged_prefill4(torch::Tensor q, torch::Tensor cache, torch::Tensor tables, torch::Tensor cu_q,
                           torch::Tensor ctx, torch::Tensor out, int64_t heads, double scale, torch::Tensor ws) {
  using namespace dsv;
  const int ng = dsv_kv4_groups(cache, "paged_prefill4");
  const int64_t hkv = cache.size(1);
  TORCH_CHECK_VALUE(heads > 0 && heads % hkv == 0 && heads / hkv <= 16,
                    "paged_prefill4: query heads must be 1 to 16 times the kv heads");
  TORCH_CHECK_VALUE(scale > 0, "paged_prefill4: scale must be positive");
  TORCH_CHECK_VALUE(q.dim() == 2 && q.size(0) < (int64_t(1) << 26), "paged_prefill4: q must be [tokens, heads * 128]");
  for (const auto* x : {&q, &out})
    TORCH_CHECK_VALUE(x->is_cuda() && x->device() == cache.device() && x->scalar_type() == at::kBFloat16 &&
                          x->dim() == 2 && x->size(0) == q.size(0) && x->size(1) == heads * HD && x->stride(1) == 1 &&
                          x->stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(x->data_ptr()) % 16 == 0,
                      "paged_prefill4: q and out must be bf16 [tokens, heads * 128] with 16-byte aligned rows on the "
                      "cache's device");
  TORCH_CHECK_VALUE(ctx.scalar_type() == at::kInt && ctx.dim() == 1 && ctx.is_contiguous() &&
                        ctx.device() == cache.device() && cu_q.scalar_type() == at::kInt && cu_q.dim() == 1 &&
                        cu_q.size(0) == ctx.size(0) + 1 && cu_q.is_contiguous() && cu_q.device() == cache.device(),
                    "paged_prefill4: cu_q must be int32 [sequences + 1], context lengths int32 [sequences]");
  TORCH_CHECK_VALUE(tables.scalar_type() == at::kInt && tables.dim() == 2 && tables.size(0) == ctx.size(0) &&
                        tables.is_contiguous() && tables.device() == cache.device(),
                    "paged_prefill4: block tables must be int32 [sequences, pages]");
  TORCH_CHECK_VALUE(tables.size(1) * cache.size(2) * 16 < (int64_t(1) << 31) && hkv < 65536,
                    "paged_prefill4: block tables of more than 2^31 tokens, or more than 65535 kv heads");
  TORCH_CHECK_VALUE(ws.is_cuda() && ws.device() == cache.device() && ws.is_contiguous() &&
                        (int64_t)ws.nbytes() >= dsv_kv4_workspace_bytes(),
                    "paged_prefill4: the workspace must come from kv4_workspace on the cache's device");
  if (q.size(0) == 0 || ctx.size(0) == 0) return 0;
  c10::cuda::CUDAGuard guard(cache.device());
  Prefill4Args a{};
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.q_stride = q.stride(0);
  a.cache = cache.data_ptr<uint8_t>();
  a.tables = tables.data_ptr<int>();
  a.cu_q = cu_q.data_ptr<int>();
  a.ctx = ctx.data_ptr<int>();
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.out_stride = out.stride(0);
  a.seqs = (int)ctx.size(0);
  a.rows = (int)q.size(0);
  a.max_pages = (int)tables.size(1);
  a.num_pages = (int)cache.size(0);
  a.kv_heads = (int)hkv;
  a.group = (int)(heads / hkv);
  a.sub = (int)cache.size(2);
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  // Two tiles per CTA share the dequantised keys; with too few of them to fill
  // the SMs, one tile per CTA.
  const int64_t all = q.size(0) * a.group;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  a.tile_rows = all / 256 * hkv >= sms ? 256 : 128;
  // With tiles for less than half of the SMs, several CTAs share a tile's keys
  // (where the tables allow a context of several key tiles at all).
  const int64_t tiles = all / a.tile_rows + a.seqs, most = (int64_t)a.max_pages * a.sub / 16;
  a.splits = (int)std::max<int64_t>(1, std::min<int64_t>(sms / (tiles * hkv), std::min<int64_t>(most, 32)));
  a.part = reinterpret_cast<float*>(ws.data_ptr());
  TORCH_CHECK(a.splits == 1 || tiles * hkv * a.splits * 128 * P4_PART * 4 <= dsv_kv4_workspace_bytes() - (1 << 20),
              "paged_prefill4: workspace too small for this GPU");
  const dim3 grid((unsigned)tiles, (unsigned)hkv, (unsigned)a.splits);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (ng == 1) prefill4_launch<1>(a, grid, stream);
  else if (ng == 2) prefill4_launch<2>(a, grid, stream);
  else prefill4_launch<4>(a, grid, stream);
  return a.splits > 1 ? 2 : 1;
}

DSV_ERROR_ACCESSOR(dsv_read_error_kv4_prefill)
