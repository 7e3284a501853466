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
// Operands are fp16 (fp32 accumulators): a value s (c + z) of the 4-bit format
// fits 11 bits to within 2^-12 of its group's range, where bf16 would double the
// result's own rounding error. K's and V's values stay below 8704 and P below
// 2^8; each query row is scaled by a power of two (its largest magnitude lands
// in [1, 2)), which the softmax undoes.
//
// K is stored as [keys x channels], V as [channels x keys] (both K-major for
// their product): the code pairs that one mask yields, channels (c, c + 4) of
// K and tokens (2t, 2t + 1) of V, are then neighbours in shared memory. For K
// the order of the eight channels of a 16-byte unit is that of the pairs
// (0, 4, 1, 5, 2, 6, 3, 7), and Q is stored in the same order.
//
// Shared memory: Q 64 KB, K 2 x 32 KB, V 2 x 32 KB. TMEM: S0, S1, O0, O1 of 128
// columns each; P_x takes the first 64 columns of S_x.
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
constexpr int P4_SMEM = 6 * P4_TILE + 1024 + 256 * 4 + 256;
constexpr float P4_LAZY = 8.f;
constexpr uint32_t P4_IDESC = (1u << 4) | (128u >> 3) << 17 | (128u >> 4) << 24;   // f16 x f16 -> f32, 128 x 128

enum : int {
  kErrP4K = 0x4401,
  kErrP4V = 0x4402,
  kErrP4S = 0x4403,
  kErrP4P = 0x4404,
  kErrP4O = 0x4405,
  kErrP4KEmpty = 0x4406,
  kErrP4VEmpty = 0x4407,
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

template <int N>
__device__ __forceinline__ void reg_grow() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_shrink() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// s (c + z) of the code pair at bits 0-3 of w's halves, after `w` was shifted
// so that the pair lies at bits 6-9: 64 + 4 c by mask, 4 c exactly, one rounding.
__device__ __forceinline__ uint32_t p4_value(uint32_t w, __half2 quarter, __half2 base) {
  const uint32_t m = (w & 0x03c003c0u) | 0x54005400u;
  const __half2 c4 = __hsub2(*reinterpret_cast<const __half2*>(&m), __float2half2_rn(64.f));
  const __half2 v = __hfma2(c4, quarter, base);
  return *reinterpret_cast<const uint32_t*>(&v);
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
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kvh = blockIdx.y;

  // Which sequence, and which of its query tiles (the last, longest first).
  int seq = -1, local = 0, left = blockIdx.x;
  for (int s0 = 0; s0 < a.seqs; s0 += 32) {
    int n = 0;
    if (s0 + lane < a.seqs) {
      const int len = a.cu_q[s0 + lane + 1] - a.cu_q[s0 + lane];
      n = len > 0 ? (len * a.group + a.tile_rows - 1) / a.tile_rows : 0;
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
      const int end = __shfl_sync(0xffffffffu, up, at);
      seq = s0 + at;
      local = end - 1 - left;
      break;
    }
    left -= __shfl_sync(0xffffffffu, up, 31);
  }
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
  const int n_max = max(n_kb[0], n_kb[1]);
  const int kv_end = pos0 + (row0 + rows - 1) / a.group + 1;

  if (threadIdx.x == 0) {
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
      const int lim = seen - j * 128;
      if (__any_sync(0xffffffffu, lim < 128)) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= lim) s[i] = -INFINITY;
      }
      float red[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) red[c] = s[c];
#pragma unroll
      for (int i = 8; i < 128; ++i) red[i & 7] = fmaxf(red[i & 7], s[i]);
      const float row_max = f * fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])),
                                      fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7])));
      // The reference maximum moves only when it is exceeded by 2^8: P stays
      // below 2^8 in fp16 and the common factor cancels in O / l.
      const bool move = m == -INFINITY || row_max > m + P4_LAZY;
      const float mx = move ? fmaxf(m, row_max) : m;
      const float corr = m == -INFINITY ? 0.f : (move ? kv4_exp2(m - mx) : 1.f);
      const float ref = mx == -INFINITY ? 0.f : mx;
      l *= corr;
      m = mx;
      // s_full of this tile was committed after the last product into O
      if (j > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(t_o + c * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * corr);
          tmem_st_32x32b_x32(t_o + c * 32, v);
        }
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float p0 = kv4_exp2(fmaf(s[c * 64 + 2 * i], f, -ref)), p1 = kv4_exp2(fmaf(s[c * 64 + 2 * i + 1], f, -ref));
          sum[(2 * i) & 3] += p0;
          sum[(2 * i + 1) & 3] += p1;
          p[i] = pack_f16(p0, p1);
        }
        tmem_st_32x32b_x32(t_s + c * 32, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[x]);
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, kv4_wait(&o_done[x], 0, kErrP4O));
    if (ok) {
      tc_fence_after();
      const float inv = l != 0.f ? 1.f / l : 0.f;           // a row that sees no key gives zeros
      __nv_bfloat16* dst = a.out + (int64_t)(q_begin + row / a.group) * a.out_stride +
                           (int64_t)(kvh * a.group + row % a.group) * HD;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(t_o + c * 32, v);
          tmem_ld_wait();
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
              w[e] = pack2_bf16(__uint_as_float(v[u * 8 + 2 * e]) * inv, __uint_as_float(v[u * 8 + 2 * e + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + c * 32 + u * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  } else if (warp < 12) {
    // -------------------------------------------------------------- dequantise
    reg_shrink<88>();
    const int w4 = warp - 8;
    const int key = w4 * 32 + lane;                        // K: this thread's key of the tile
    const int g = lane >> 2, t = lane & 3;
    auto record = [&](int rec) -> const uint8_t* {          // K record of 16-token block `rec`; null past the end
      if (rec * 16 >= kv_end) return nullptr;
      const int page = tab[rec / a.sub];
      if ((unsigned)page >= (unsigned)a.num_pages) {
        set_error(kErrShape);
        return nullptr;
      }
      return a.cache + (((size_t)page * a.kv_heads + kvh) * a.sub + rec % a.sub) * (2 * kv4_record(NG));
    };
    uint4 kc[4], vc[2][2];
    uint32_t kp[NG];
    const uint8_t* vrec[2];
    auto load_k = [&](int j) {
      const uint8_t* p = record(j * 8 + key / 16);
      if (p != nullptr && j * 128 + key >= kv_end) p = nullptr;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        kc[i] = p != nullptr ? *reinterpret_cast<const uint4*>(p + (key & 15) * 64 + i * 16) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NG; ++i)
        kp[i] = p != nullptr ? *reinterpret_cast<const uint32_t*>(p + KV4_CODES + 64 * i + 4 * (key & 15)) : 0u;
    };
    auto load_v = [&](int j) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        vrec[b] = record(j * 8 + w4 * 2 + b);
        if (vrec[b] != nullptr) vrec[b] += kv4_record(NG);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          vc[b][i] = vrec[b] != nullptr ? *reinterpret_cast<const uint4*>(vrec[b] + i * 512 + lane * 16) : make_uint4(0, 0, 0, 0);
      }
    };
    if (n_max > 0) {
      load_k(0);
      load_v(0);
    }
    for (int j = 0; j < n_max; ++j) {
      const int st = j & 1;
      const uint32_t ph = ((uint32_t)(j >> 1) & 1u) ^ 1u;
      if (!__all_sync(0xffffffffu, kv4_wait(&k_empty[st], ph, kErrP4KEmpty))) break;
      {
        uint8_t* dst = sK + st * P4_TILE + key * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {                       // 16-byte words of lane t = i: word e covers channels 32 e + 8 i
          const uint32_t x[4] = {kc[i].x, kc[i].y, kc[i].z, kc[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t pw = kp[e * NG / 4];
            const __half2 quarter = __float2half2_rn(kv4_scale(pw) * 0.25f);
            const __half2 base = __float2half2_rn(kv4_scale(pw) * kv4_zero(pw));
            const int u = 4 * e + i;                        // 16-byte unit of the row
            *reinterpret_cast<uint4*>(dst + (u >> 3) * P4_CHUNK + (((u & 7) ^ (key & 7)) << 4)) =
                make_uint4(p4_value(x[e] << 6, quarter, base), p4_value(x[e] << 2, quarter, base),
                           p4_value(x[e] >> 2, quarter, base), p4_value(x[e] >> 6, quarter, base));
          }
        }
      }
      if (j + 1 < n_max) load_k(j + 1);
      fence_proxy_async_smem();
      mbar_arrive(&k_full[st]);
      if (!__all_sync(0xffffffffu, kv4_wait(&v_empty[st], ph, kErrP4VEmpty))) break;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int rec = w4 * 2 + b;
        const int tok = j * 128 + rec * 16 + 2 * t;         // tokens tok, tok + 1, tok + 8, tok + 9
        uint8_t* dst = sV + st * P4_TILE + (rec >> 2) * P4_CHUNK + g * 128 + 4 * t;
        const int u = 2 * (rec & 3);                        // 16-byte unit (8 tokens) of the row; u + 1 the late half
        const uint32_t x[8] = {vc[b][0].x, vc[b][0].y, vc[b][0].z, vc[b][0].w,
                               vc[b][1].x, vc[b][1].y, vc[b][1].z, vc[b][1].w};
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          __half2 quarter[2], base[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint2 pw = make_uint2(0, 0);
            if (vrec[b] != nullptr) pw = *reinterpret_cast<const uint2*>(vrec[b] + KV4_CODES + 64 * i + 8 * t + 32 * h);
            // a key that no query sees is a zero row whatever its record holds
            if (tok + 8 * h >= kv_end) pw.x = 0;
            if (tok + 8 * h + 1 >= kv_end) pw.y = 0;
            const float s0 = kv4_scale(pw.x), s1 = kv4_scale(pw.y);
            quarter[h] = __floats2half2_rn(s0 * 0.25f, s1 * 0.25f);
            base[h] = __floats2half2_rn(s0 * kv4_zero(pw.x), s1 * kv4_zero(pw.y));
          }
#pragma unroll
          for (int q = 0; q < 8 / NG; ++q) {
            const int mt = i * (8 / NG) + q;                // channels 16 mt + g and + 8
            uint8_t* d0 = dst + mt * 2048;
            *reinterpret_cast<uint32_t*>(d0 + ((u ^ g) << 4)) = p4_value(x[mt] << 6, quarter[0], base[0]);
            *reinterpret_cast<uint32_t*>(d0 + 1024 + ((u ^ g) << 4)) = p4_value(x[mt] << 2, quarter[0], base[0]);
            *reinterpret_cast<uint32_t*>(d0 + (((u + 1) ^ g) << 4)) = p4_value(x[mt] >> 2, quarter[1], base[1]);
            *reinterpret_cast<uint32_t*>(d0 + 1024 + (((u + 1) ^ g) << 4)) = p4_value(x[mt] >> 6, quarter[1], base[1]);
          }
        }
      }
      if (j + 1 < n_max) load_v(j + 1);
      fence_proxy_async_smem();
      mbar_arrive(&v_full[st]);
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

template <int NG>
static void prefill4_launch(const Prefill4Args& a, dim3 grid, cudaStream_t stream) {
  static const cudaError_t attr =
      cudaFuncSetAttribute(prefill4_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, P4_SMEM);
  C10_CUDA_CHECK(attr);
  prefill4_kernel<NG><<<grid, P4_THREADS, P4_SMEM, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
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
  a.tile_rows = all / 256 * hkv >= at::cuda::getCurrentDeviceProperties()->multiProcessorCount ? 256 : 128;
  const dim3 grid((unsigned)(all / a.tile_rows + a.seqs), (unsigned)hkv);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (ng == 1) prefill4_launch<1>(a, grid, stream);
  else if (ng == 2) prefill4_launch<2>(a, grid, stream);
  else prefill4_launch<4>(a, grid, stream);
  return 1;
}

DSV_ERROR_ACCESSOR(dsv_read_error_kv4_prefill)
