// Writing, reading and copying the 4-bit KV cache (format: kv4.cuh).
//
// The reference project keeps its cache in the serving library's bf16 pages and
// has no counterpart of these kernels.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "kv4.cuh"

namespace dsv {

// Rows x heads from which records are assembled. One by one against by records, us:
//   rows x heads   1 head        2 heads       8 heads
//    8192           5.5 /  7.4    5.7 /  7.8    5.7 /  7.5
//   16384           9.3 / 10.5    9.4 / 10.9    9.7 /  9.2
//   32768          16.8 / 15.2   16.8 / 15.4   17.0 / 14.2
//   65536          31.2 / 25.1   31.2 / 25.0   31.2 / 23.4
constexpr int64_t KV4_MANY = 32768;

struct Kv4RowsArgs {
  const __nv_bfloat16* k;   // [T, Hkv, 128], strides in elements
  const __nv_bfloat16* v;
  int64_t k_row, k_head, v_row, v_head;
  uint8_t* cache;
  const int64_t* slots;     // [T], negative = not cached
  int64_t num_slots;        // pages * page size
  int rows, heads, page;
  __nv_bfloat16* k_out;     // read: contiguous [T, Hkv * 128]
  __nv_bfloat16* v_out;
};

// Address of the K record of a slot's token and head, and the token's place in it.
template <int NG>
__device__ __forceinline__ uint8_t* kv4_record_of(const Kv4RowsArgs& a, int64_t slot, int head, int& r) {
  const int64_t page = slot / a.page;
  const int off = (int)(slot - page * a.page);
  r = off & 15;
  return a.cache + (size_t)(((page * a.heads + head) * (a.page / 16) + (off >> 4)) * 2) * kv4_record(NG);
}

__device__ __forceinline__ float nan_min(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float nan_max(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Quantising this lane's 4 channels (4 lane .. + 3) of a row, in three steps.
// Each is rounded as the format says (no contraction), so any implementation of
// it gives these bits.
//
// The group's range; the 32 / NG lanes that share the group all get it.
template <int NG>
__device__ __forceinline__ void kv4_range(float (&x)[4], float& lo, float& hi) {
  lo = nan_min(nan_min(x[0], x[1]), nan_min(x[2], x[3]));
  hi = nan_max(nan_max(x[0], x[1]), nan_max(x[2], x[3]));
  if (__any_sync(0xffffffffu, !(lo >= -KV4_LIMIT && hi <= KV4_LIMIT))) {       // saturate; a NaN counts as 0
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = x[e] == x[e] ? fminf(fmaxf(x[e], -KV4_LIMIT), KV4_LIMIT) : 0.f;
    lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
    hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  }
  lo = fminf(lo, 0.f);
  hi = fmaxf(hi, 0.f);
#pragma unroll
  for (int o = 1; o < 32 / NG; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
}
// Its (scale, zero point) word and the scale's reciprocal.
__device__ __forceinline__ uint32_t kv4_word(float lo, float hi, float& inv) {
  float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
  if (s < KV4_TINY) s = 0.f;
  inv = s > 0.f ? __frcp_rn(s) : 0.f;
  return __float_as_uint(s) | __half_as_ushort(__float2half_rn(__fmul_rn(lo, inv)));
}
// The four codes as nibbles. In [0, 15] adding 1.5 * 2^23 rounds to the nearest
// integer (ties to even) and leaves it in the low bits.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[4], uint32_t word, float inv) {
  const float z = kv4_zero(word);
  uint32_t u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    u[e] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fsub_rn(__fmul_rn(x[e], inv), z), 0.f), 15.f), 12582912.f));
  return (u[0] + (u[1] << 4) + (u[2] << 8) + (u[3] << 12)) & 0xffffu;
}

// Code e of four nibbles as a float, exactly: 2^23 + c by its bits, minus 2^23.
__device__ __forceinline__ float kv4_code(uint32_t codes, int e) {
  return __uint_as_float(0x4b000000u | (codes >> (4 * e) & 15u)) - 8388608.f;
}

__device__ __forceinline__ void kv4_load4(const __nv_bfloat16* p, bool vec, float (&x)[4]) {
  if (vec) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    x[0] = __uint_as_float(w.x << 16);
    x[1] = __uint_as_float(w.x & 0xffff0000u);
    x[2] = __uint_as_float(w.y << 16);
    x[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = bf2f(p[e]);
  }
}

// This lane's 4 channels of a row's K and V of one head.
__device__ __forceinline__ void kv4_load_row(const Kv4RowsArgs& a, bool vec, int row, int head, float (&x)[4],
                                             float (&y)[4]) {
  const int c = 4 * (threadIdx.x & 31);
  kv4_load4(a.k + row * a.k_row + head * a.k_head + c, vec, x);
  kv4_load4(a.v + row * a.v_row + head * a.v_head + c, vec, y);
}

// Codes and word of token r of a record's K or V part (shared or global memory).
template <int NG>
__device__ __forceinline__ void kv4_put_k(uint8_t* krec, int r, uint32_t c, uint32_t word) {
  const int lane = threadIdx.x & 31;
  // lane's codes are half a word of channels 32 i + 8 t + 0..7
  const uint32_t up = __shfl_down_sync(0xffffffffu, c, 1);
  if (!(lane & 1))
    *reinterpret_cast<uint32_t*>(krec + 64 * r + 16 * (lane % 8 / 2) + 4 * (lane / 8)) = c | up << 16;
  if (lane % (32 / NG) == 0)
    *reinterpret_cast<uint32_t*>(krec + KV4_CODES + 64 * (lane * NG / 32) + 4 * r) = word;
}
template <int NG>
__device__ __forceinline__ void kv4_put_v(uint8_t* vrec, int r, uint32_t c, uint32_t word) {
  const int lane = threadIdx.x & 31;
  // channels g and g + 8 of a 16-channel tile share a byte; lane ^ 2 holds the other half
  const uint32_t hi = __shfl_down_sync(0xffffffffu, c, 2);
  if (!(lane & 2)) {
    uint8_t* dst = vrec + 512 * (lane / 16) + 16 * (r % 8 / 2) + 4 * (lane / 4 % 4) + (r / 8) + 2 * (r % 2);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      dst[64 * (4 * (lane & 1) + e)] = (uint8_t)((c >> (4 * e) & 15u) | (hi >> (4 * e) & 15u) << 4);
  }
  if (lane % (32 / NG) == 0)
    *reinterpret_cast<uint32_t*>(vrec + KV4_CODES + 64 * (lane * NG / 32) + 4 * r) = word;
}

// One row's K and V into token r of the record at `krec`.
template <int NG>
__device__ __forceinline__ void kv4_put_row(float (&x)[4], float (&y)[4], uint8_t* krec, int r) {
  float lo, hi, inv;
  kv4_range<NG>(x, lo, hi);
  uint32_t word = kv4_word(lo, hi, inv);
  kv4_put_k<NG>(krec, r, kv4_codes(x, word, inv), word);
  kv4_range<NG>(y, lo, hi);
  word = kv4_word(lo, hi, inv);
  kv4_put_v<NG>(krec + kv4_record(NG), r, kv4_codes(y, word, inv), word);
}

// Four rows' words at once: their 8 NG groups (K and V) take one lane each, so
// that the two exact divisions run once and not eight times. put(j, c, word,
// d, word) stores row j's K and V.
template <int NG, class Put>
__device__ __forceinline__ void kv4_four_rows(float (&x)[4][4], float (&y)[4][4], Put put) {
  const int lane = threadIdx.x & 31;
  float lo[8], hi[8], mylo = 0.f, myhi = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kv4_range<NG>(x[j], lo[2 * j], hi[2 * j]);
    kv4_range<NG>(y[j], lo[2 * j + 1], hi[2 * j + 1]);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {                // lane 8 i + k takes group i of item k
    const float a = __shfl_sync(0xffffffffu, lo[k], (lane >> 3) % NG * (32 / NG));
    const float b = __shfl_sync(0xffffffffu, hi[k], (lane >> 3) % NG * (32 / NG));
    if ((lane & 7) == k) {
      mylo = a;
      myhi = b;
    }
  }
  float inv;
  const uint32_t word = kv4_word(mylo, myhi, inv);
  const int from = 8 * (lane * NG / 32);       // this lane's own group
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t kw = __shfl_sync(0xffffffffu, word, from + 2 * j), vw = __shfl_sync(0xffffffffu, word, from + 2 * j + 1);
    const float ki = __shfl_sync(0xffffffffu, inv, from + 2 * j), vi = __shfl_sync(0xffffffffu, inv, from + 2 * j + 1);
    put(j, kv4_codes(x[j], kw, ki), kw, kv4_codes(y[j], vw, vi), vw);
  }
}

// The values of token r of a record (null: zeros) as bf16 rows.
template <int NG>
__device__ __forceinline__ void kv4_get_row(const Kv4RowsArgs& a, int row, int head, const uint8_t* krec, int r) {
  const int lane = threadIdx.x & 31;
  uint2 ko = make_uint2(0, 0), vo = make_uint2(0, 0);
  if (krec != nullptr) {
    const uint8_t* vrec = krec + kv4_record(NG);
    const uint32_t kc =
        *reinterpret_cast<const uint16_t*>(krec + 64 * r + 16 * (lane % 8 / 2) + 4 * (lane / 8) + 2 * (lane & 1));
    const uint8_t* src = vrec + 512 * (lane / 16) + 16 * (r % 8 / 2) + 4 * (lane / 4 % 4) + (r / 8) + 2 * (r % 2);
    uint32_t vc = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) vc |= ((uint32_t)src[64 * (4 * (lane & 1) + e)] >> (lane & 2 ? 4 : 0) & 15u) << (4 * e);
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(krec + KV4_CODES + 64 * (lane * NG / 32) + 4 * r);
    const uint32_t vw = *reinterpret_cast<const uint32_t*>(vrec + KV4_CODES + 64 * (lane * NG / 32) + 4 * r);
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = kv4_scale(kw) * (kv4_code(kc, e) + kv4_zero(kw));
      y[e] = kv4_scale(vw) * (kv4_code(vc, e) + kv4_zero(vw));
    }
    ko = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
    vo = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
  }
  const size_t at = ((size_t)row * a.heads + head) * HD + 4 * lane;
  *reinterpret_cast<uint2*>(a.k_out + at) = ko;
  *reinterpret_cast<uint2*>(a.v_out + at) = vo;
}

// One warp = one (row, head), K and V: 64 rows of 8 heads are written in 2.8 us
// and read in 2.3 us, 8192 read in 18 us (6.6 us of HBM bytes; the single-byte
// V accesses and their partial sectors are what it waits for).
template <int NG, bool WRITE>
__global__ void __launch_bounds__(256) kv4_row_kernel(const Kv4RowsArgs a, bool vec) {
  const int64_t w = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 32;
  if (w >= (int64_t)a.rows * a.heads) return;
  const int row = (int)(w / a.heads), head = (int)(w % a.heads);
  int64_t slot = a.slots[row];
  if (slot >= a.num_slots) {
    if ((threadIdx.x & 31) == 0) set_error(kErrShape);
    slot = -1;
  }
  int r = 0;
  uint8_t* krec = slot >= 0 ? kv4_record_of<NG>(a, slot, head, r) : nullptr;
  if (!WRITE) kv4_get_row<NG>(a, row, head, krec, r);
  else if (krec != nullptr) {
    float x[4], y[4];
    kv4_load_row(a, vec, row, head, x, y);
    kv4_put_row<NG>(x, y, krec, r);
  }
}

// Writing many rows: four warps = 16 rows of one head. Where 16 rows that follow
// one another fill a record (most of a prompt), the record is assembled in
// shared memory and stored as one run of 16-byte accesses: a lone token's V codes
// are 64 bytes in 16 sectors, and those partial sectors bound the row-by-row
// kernel (32 us for 8192 rows of 8 heads, whatever its instruction count). The
// record belongs to the warps whose rows it begins in; rows outside such records
// go one by one. A row's quantisation is a chain of about a microsecond (two
// statistics across lanes, two exact divisions): hence four rows per warp, whose
// divisions share a pass. 8192 rows of 8 heads: 25 us (16 rows per warp: 36 us).
template <int NG>
__global__ void __launch_bounds__(256) kv4_write_records_kernel(const Kv4RowsArgs a, bool vec) {
  constexpr int REC = 2 * kv4_record(NG);
  __shared__ __align__(16) uint8_t records[2][REC];
  const int lane = threadIdx.x & 31, team = threadIdx.x / 128, part = threadIdx.x / 32 & 3;
  uint8_t* rec = records[team];
  const int64_t w = (int64_t)blockIdx.x * 2 + team;
  const int head = (int)(w % a.heads), row0 = (int)(w / a.heads) * 16;
  if (row0 >= a.rows) return;                 // the whole team
  // Window of 48 rows from 16 before ours: bit j of `run`: row j + 1's slot is
  // the next one; of `begins`: row j's slot begins a record that 16 rows fill.
  auto slot_of = [&](int row) { return row >= 0 && row < a.rows ? a.slots[row] : (int64_t)-1; };
  const int64_t s0 = slot_of(row0 - 16 + lane), s1 = slot_of(row0 + 16 + lane);
  const int64_t n0 = __shfl_down_sync(0xffffffffu, s0, 1), n1 = __shfl_down_sync(0xffffffffu, s1, 1);
  const int64_t first1 = __shfl_sync(0xffffffffu, s1, 0);
  const bool f0 = s0 >= 0 && (lane == 31 ? first1 : n0) == s0 + 1, f1 = s1 >= 0 && lane < 31 && n1 == s1 + 1;
  const bool b0 = s0 >= 0 && (s0 & 15) == 0 && s0 + 15 < a.num_slots;
  const bool b1 = s1 >= 0 && (s1 & 15) == 0 && s1 + 15 < a.num_slots;
  uint64_t run = __ballot_sync(0xffffffffu, f0) | (uint64_t)__ballot_sync(0xffffffffu, f1) << 32;
  run &= run >> 1;
  run &= run >> 2;
  run &= run >> 4;                            // eight steps in a row
  run &= run >> 7;                            // fifteen
  const uint64_t begins = run & (__ballot_sync(0xffffffffu, b0) | (uint64_t)__ballot_sync(0xffffffffu, b1) << 32);
  uint64_t whole = begins;                    // rows of whole records
  whole |= whole << 1;
  whole |= whole << 2;
  whole |= whole << 4;
  whole |= whole << 8;
  const uint32_t mine = (uint32_t)(begins >> 16) & 0xffffu;
  if (mine != 0) {
    const int row = row0 + __ffs(mine) - 1;
    int r;
    uint8_t* dst = kv4_record_of<NG>(a, a.slots[row], head, r);
    float x[4][4], y[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) kv4_load_row(a, vec, row + 4 * part + j, head, x[j], y[j]);
    kv4_four_rows<NG>(x, y, [&](int j, uint32_t kc, uint32_t kw, uint32_t vc, uint32_t vw) {
      kv4_put_k<NG>(rec, 4 * part + j, kc, kw);
      kv4_put_v<NG>(rec + kv4_record(NG), 4 * part + j, vc, vw);
    });
    named_bar_sync(1 + team, 128);
    for (int i = threadIdx.x & 127; i < REC / 16; i += 128)
      reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(rec)[i];
  }
  // The rest of this warp's four rows.
  const bool own = lane < 16 ? false : s0 >= 0 && !(whole >> lane & 1u);       // window rows 16..31 are ours
  if (own && s0 >= a.num_slots) set_error(kErrShape);
  const uint32_t rest = __ballot_sync(0xffffffffu, own && s0 < a.num_slots) >> 16;
  if (!(rest >> (4 * part) & 15u)) return;
  float x[4][4], y[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) kv4_load_row(a, vec, min(row0 + 4 * part + j, a.rows - 1), head, x[j], y[j]);
  kv4_four_rows<NG>(x, y, [&](int j, uint32_t kc, uint32_t kw, uint32_t vc, uint32_t vw) {
    const int64_t slot = __shfl_sync(0xffffffffu, s0, 16 + 4 * part + j);
    if (!(rest >> (4 * part + j) & 1u)) return;
    int r;
    uint8_t* krec = kv4_record_of<NG>(a, slot, head, r);
    kv4_put_k<NG>(krec, r, kc, kw);
    kv4_put_v<NG>(krec + kv4_record(NG), r, vc, vw);
  });
}

template <bool WRITE>
static void kv4_rows_launch(const Kv4RowsArgs& a, bool vec, int ng) {
  if (a.rows == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (WRITE && (int64_t)a.rows * a.heads >= KV4_MANY) {
    const int64_t teams = (int64_t)((a.rows + 15) / 16) * a.heads;
    auto kernel = ng == 1 ? kv4_write_records_kernel<1> : ng == 2 ? kv4_write_records_kernel<2> : kv4_write_records_kernel<4>;
    kernel<<<(unsigned)((teams + 1) / 2), 256, 0, stream>>>(a, vec);
  } else {
    const int64_t warps = (int64_t)a.rows * a.heads;
    auto kernel = ng == 1 ? kv4_row_kernel<1, WRITE> : ng == 2 ? kv4_row_kernel<2, WRITE> : kv4_row_kernel<4, WRITE>;
    kernel<<<(unsigned)((warps + 7) / 8), 256, 0, stream>>>(a, vec);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// ------------------------------------------------------------------ page copies

constexpr int CP_TENSORS = 192;   // caches per launch
constexpr int CP_PAIRS = 512;     // pages per launch
constexpr int CP_THREADS = 256;
constexpr int CP_UNITS = 4;       // 16-byte units per thread: a CTA moves 16 KB

// Pages and addresses travel in the launch's arguments: no copy to the device,
// nothing to keep alive until the kernel has read it.
struct CopyPagesArgs {
  uint8_t* base[CP_TENSORS];
  int2 pair[CP_PAIRS];      // (source, destination)
  int64_t page_units;       // 16-byte units per page
  int pairs, chunks;        // chunks: CTAs per page
};

// grid (chunk + chunks * pair, tensor).
__global__ void __launch_bounds__(CP_THREADS) copy_pages_kernel(const __grid_constant__ CopyPagesArgs a) {
  const int p = blockIdx.x / a.chunks;
  const int64_t u0 = (int64_t)(blockIdx.x - p * a.chunks) * (CP_THREADS * CP_UNITS) + threadIdx.x;
  uint8_t* base = a.base[blockIdx.y];
  const uint4* src = reinterpret_cast<const uint4*>(base) + a.pair[p].x * a.page_units;
  uint4* dst = reinterpret_cast<uint4*>(base) + a.pair[p].y * a.page_units;
  uint4 v[CP_UNITS];
#pragma unroll
  for (int i = 0; i < CP_UNITS; ++i)
    if (u0 + i * CP_THREADS < a.page_units) v[i] = __ldcs(src + u0 + i * CP_THREADS);
#pragma unroll
  for (int i = 0; i < CP_UNITS; ++i)
    if (u0 + i * CP_THREADS < a.page_units) __stcs(dst + u0 + i * CP_THREADS, v[i]);
}

}  // namespace dsv

// ---------------------------------------------------------------- bindings

// Checks a 4-bit cache and returns its number of groups per row. (Numbers enter
// these messages as strings: formatting one through a stream crashed in a process
// whose CUDA driver was loaded.)
int dsv_kv4_groups(const torch::Tensor& cache, const char* op) {
  TORCH_CHECK_VALUE(cache.is_cuda() && cache.scalar_type() == at::kByte && cache.dim() == 5 && cache.size(3) == 2,
                    op, ": cache must be a CUDA uint8 tensor [pages, kv heads, page size / 16, 2, record bytes]");
  TORCH_CHECK_VALUE(cache.is_contiguous() && reinterpret_cast<uintptr_t>(cache.data_ptr()) % 16 == 0, op,
                    ": cache must be contiguous and 16-byte aligned");
  TORCH_CHECK_VALUE(cache.size(0) > 0 && cache.size(1) > 0 && cache.size(2) > 0, op,
                    ": cache has no pages, no kv heads or no 16-token records");
  const int64_t rec = cache.size(4);
  const int ng = rec == dsv::kv4_record(1) ? 1 : rec == dsv::kv4_record(2) ? 2 : rec == dsv::kv4_record(4) ? 4 : 0;
  TORCH_CHECK_VALUE(ng != 0, op, ": record of ", std::to_string(rec), " bytes is none of 1088, 1152, 1280 (groups of 128, 64, 32)");
  return ng;
}

static void kv4_rows(const char* op, const torch::Tensor& x, int heads, int64_t rows, int64_t& row, int64_t& head,
                     bool& vec) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.scalar_type() == at::kBFloat16, op, ": k and v must be bf16 CUDA tensors");
  const bool flat = x.dim() == 2;
  TORCH_CHECK_VALUE(flat ? x.size(1) == (int64_t)heads * dsv::HD
                         : x.dim() == 3 && x.size(1) == heads && x.size(2) == dsv::HD,
                    op, ": k and v must be [rows, kv heads * 128] or [rows, kv heads, 128]");
  TORCH_CHECK_VALUE(x.size(0) == rows && x.stride(-1) == 1, op, ": k, v and slots must have the same rows, contiguous along the channels");
  row = x.stride(0);
  head = flat ? dsv::HD : x.stride(1);
  vec = vec && row % 4 == 0 && head % 4 == 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 8 == 0;
}

static dsv::Kv4RowsArgs kv4_rows_args(const char* op, const torch::Tensor& cache, const torch::Tensor& slots) {
  TORCH_CHECK_VALUE(slots.is_cuda() && slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous() &&
                        slots.device() == cache.device(),
                    op, ": slots must be a contiguous int64 vector on the cache's device");
  TORCH_CHECK_VALUE(slots.size(0) < (int64_t(1) << 31), op, ": too many rows");
  dsv::Kv4RowsArgs a{};
  a.cache = cache.data_ptr<uint8_t>();
  a.slots = slots.data_ptr<int64_t>();
  a.rows = (int)slots.size(0);
  a.heads = (int)cache.size(1);
  a.page = (int)cache.size(2) * 16;
  a.num_slots = cache.size(0) * a.page;
  return a;
}

void dsv_kv4_write(torch::Tensor k, torch::Tensor v, torch::Tensor cache, torch::Tensor slots) {
  using namespace dsv;
  const int ng = dsv_kv4_groups(cache, "kv4_write");
  Kv4RowsArgs a = kv4_rows_args("kv4_write", cache, slots);
  bool vec = true;
  kv4_rows("kv4_write", k, a.heads, a.rows, a.k_row, a.k_head, vec);
  kv4_rows("kv4_write", v, a.heads, a.rows, a.v_row, a.v_head, vec);
  TORCH_CHECK_VALUE(k.device() == cache.device() && v.device() == cache.device(),
                    "kv4_write: k, v and the cache must be on one device");
  a.k = reinterpret_cast<const __nv_bfloat16*>(k.data_ptr());
  a.v = reinterpret_cast<const __nv_bfloat16*>(v.data_ptr());
  c10::cuda::CUDAGuard guard(cache.device());
  kv4_rows_launch<true>(a, vec, ng);
}

std::tuple<torch::Tensor, torch::Tensor> dsv_kv4_read(torch::Tensor cache, torch::Tensor slots) {
  using namespace dsv;
  const int ng = dsv_kv4_groups(cache, "kv4_read");
  Kv4RowsArgs a = kv4_rows_args("kv4_read", cache, slots);
  c10::cuda::CUDAGuard guard(cache.device());
  auto opt = cache.options().dtype(at::kBFloat16);
  torch::Tensor k = torch::empty({a.rows, (int64_t)a.heads * HD}, opt), v = torch::empty_like(k);
  a.k_out = reinterpret_cast<__nv_bfloat16*>(k.data_ptr());
  a.v_out = reinterpret_cast<__nv_bfloat16*>(v.data_ptr());
  kv4_rows_launch<false>(a, true, ng);
  return {k, v};
}

// Returns the number of kernels launched.
int64_t dsv_copy_pages(std::vector<torch::Tensor> caches, std::vector<int64_t> src, std::vector<int64_t> dst) {
  using namespace dsv;
  if (caches.empty() || src.empty()) return 0;
  const torch::Tensor& c0 = caches[0];
  const int64_t pages = c0.size(0);
  const int64_t bytes = pages > 0 ? (int64_t)c0.nbytes() / pages : 0;
  for (const auto& c : caches) {
    TORCH_CHECK_VALUE(c.is_cuda() && c.device() == c0.device() && c.is_contiguous() && c.dim() >= 1 &&
                          c.size(0) == pages && (int64_t)c.nbytes() == pages * bytes,
                      "copy_pages: caches must be contiguous tensors of one shape and element size on one device");
    TORCH_CHECK_VALUE(reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0,
                      "copy_pages: caches must be 16-byte aligned");
  }
  TORCH_CHECK_VALUE(bytes % 16 == 0, "copy_pages: a page must be a multiple of 16 bytes");
  if (bytes == 0) return 0;
  c10::cuda::CUDAGuard guard(c0.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  CopyPagesArgs a;
  a.page_units = bytes / 16;
  const int64_t chunks = (a.page_units + CP_THREADS * CP_UNITS - 1) / (CP_THREADS * CP_UNITS);
  TORCH_CHECK_VALUE(chunks * CP_PAIRS < (int64_t(1) << 31), "copy_pages: page too large");
  a.chunks = (int)chunks;
  int64_t launches = 0;
  for (size_t t0 = 0; t0 < caches.size(); t0 += CP_TENSORS) {
    const int nt = (int)std::min<size_t>(CP_TENSORS, caches.size() - t0);
    for (int i = 0; i < nt; ++i) a.base[i] = reinterpret_cast<uint8_t*>(caches[t0 + i].data_ptr());
    for (size_t p0 = 0; p0 < src.size(); p0 += CP_PAIRS) {
      a.pairs = (int)std::min<size_t>(CP_PAIRS, src.size() - p0);
      for (int i = 0; i < a.pairs; ++i) a.pair[i] = make_int2((int)src[p0 + i], (int)dst[p0 + i]);
      copy_pages_kernel<<<dim3((unsigned)(a.pairs * a.chunks), (unsigned)nt), CP_THREADS, 0, stream>>>(a);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      ++launches;
    }
  }
  return launches;
}

DSV_ERROR_ACCESSOR(dsv_read_error_kv4_cache)
