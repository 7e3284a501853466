// Decode attention over the 4-bit paged KV cache (format and tile arithmetic:
// kv4.cuh): one query token per sequence, grouped heads, fp32 softmax.
//
// The reference project decodes over its serving library's bf16 pages; this is
// the same function over the values the codes stand for.
//
// The work is the list of 32-token pieces (two records) of every (sequence, KV head),
// cut into equal runs, one per resident warp, from the lengths on the device:
// uneven contexts share the SMs evenly and a captured launch serves any lengths.
// Warps are independent: each streams its run through a ring of bulk copies of
// its own, ahead across segments, so the loop has no barrier but the copy's. The
// GQA group's query heads are the columns of the matrix tiles and share every
// byte read.
//
// A segment that lies in one run is written by its warp. Otherwise each of its
// runs leaves a partial result in the workspace and the last to arrive joins
// them: by eights, in a tree over the runs' numbers, so that a context spread
// over the whole GPU takes four short joins and the result does not depend on
// the order of arrival.
//
// Measured against the HBM time of the cache bytes (6.54 TB/s): batch 200 x 4096,
// 32 / 8 heads, groups of 64: 184 us, 5.2 TB/s (one record per step in place of
// two was a sixth slower); 16 x 32768, 64 / 8 heads, groups of 128: 114 us in a
// graph, 5.0 TB/s. There about 240 instructions per 16 tokens and their latencies
// bound it (issue slots and ALU 53 % busy, matrix instructions 29 %). Short
// contexts are bound by a segment's fixed chain of about 2 us (queries, last
// partial sums, store) and a join's 3 us (release, counter, two rounds of loads).
// At least two pieces a run: 1 measured 9.9, 2 7.6 and 4 10.5 us at 64 x 64 tokens.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "kv4.cuh"

int dsv_kv4_groups(const torch::Tensor& cache, const char* op);

namespace dsv {

constexpr int D4_WARPS = 4;                  // per CTA
constexpr int D4_MAX_STAGES = 16;
constexpr int D4_PAGES = 32;                 // page ids looked up at a time: one per record of 16 pieces
constexpr int D4_LEVELS = 5;                 // 8^4 runs at most, and the last join's own level

enum : int {
  kErrD4Full = 0x4301,
};

// The workspace: the attention kernels' partial results, then the decode
// kernel's arrival counters.
constexpr int64_t WS_PARTS = 24 << 20;
constexpr int D4_MAX_RUNS = 4096;

struct Decode4Args {
  const __nv_bfloat16* q;   // [B, Hq * 128], row stride q_stride
  int64_t q_stride;
  const uint8_t* cache;
  const int* tables;        // [B, max_pages]
  const int* ctx;           // [B]
  __nv_bfloat16* out;       // [B, Hq * 128], row stride out_stride
  int64_t out_stride;
  bool out_vec;             // out rows are 4-byte aligned
  float4* part;             // [runs, 2, Kv4Warp::PART]
  int* arrived;             // [D4_LEVELS][runs, 2], zero between calls
  int batch, max_pages, num_pages, heads, kv_heads, group, sub;   // sub: records per page
  int stages, min_run;      // ring depth; fewest pieces of a run
  float scale_log2;
};

__device__ __forceinline__ int atom_add_acq_rel(int* p, int v) {
  int old;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], %2;" : "=r"(old) : "l"(p), "r"(v) : "memory");
  return old;
}

// A position in the list of pieces: sequence, KV head, piece; sequences without
// context have none.
struct D4Cursor {
  int b, h, c, n, len;      // n: pieces of sequence b; len: its context
  __device__ __forceinline__ void load(const Decode4Args& a) {
    len = min(a.ctx[b], a.max_pages * a.sub * 16);
    n = len > 0 ? (len + 31) / 32 : 0;
  }
  __device__ __forceinline__ void advance(const Decode4Args& a, int by) {
    c += by;
    while (c >= n) {
      c -= n;
      if (n == 0 || ++h == a.kv_heads) {
        h = 0;
        if (++b >= a.batch) {                // past the end: nothing follows
          b = a.batch - 1;
          n = 0x7fffffff;
          c = 0;
          return;
        }
        load(a);
      }
    }
  }
};

__device__ __forceinline__ int d4_pieces(const Decode4Args& a, int b) {
  return b < a.batch ? (max(0, min(a.ctx[b], a.max_pages * a.sub * 16)) + 31) / 32 : 0;
}
__device__ __forceinline__ int d4_total(const Decode4Args& a) {
  int sum = 0;
  for (int b = threadIdx.x & 31; b < a.batch; b += 32) sum += d4_pieces(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum * a.kv_heads;
}
// The cursor at piece `at` of the list.
__device__ __forceinline__ D4Cursor d4_at(const Decode4Args& a, int at) {
  const int lane = threadIdx.x & 31;
  D4Cursor w{0, 0, 0, 0, 0};
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int n = d4_pieces(a, b0 + lane) * a.kv_heads;
    int up = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, up > at);
    if (past != 0) {
      const int src = __ffs(past) - 1;
      w.b = b0 + src;
      at -= __shfl_sync(0xffffffffu, up - n, src);
      break;
    }
    at -= __shfl_sync(0xffffffffu, up, 31);
  }
  w.load(a);
  w.h = at / w.n;
  w.c = at - w.h * w.n;
  return w;
}

template <int NG, int NH, int MIN_CTAS>
__global__ void __launch_bounds__(D4_WARPS * 32, MIN_CTAS) decode4_kernel(const Decode4Args a) {
  extern __shared__ __align__(128) uint8_t d4_smem[];
  constexpr int REC = 2 * kv4_record(NG);    // K and V of 16 tokens
  using Warp = Kv4Warp<NG, NH>;
  __shared__ uint64_t full_bars[D4_WARPS][D4_MAX_STAGES];
  __shared__ int page_ids[D4_WARPS][D4_PAGES];
  __shared__ float rs[D4_WARPS][NG];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  uint8_t* ring = d4_smem + warp * a.stages * (2 * REC);
  uint64_t* full = full_bars[warp];
  int* pages = page_ids[warp];

  // Sequences without context give zeros; one longer than its table is an error
  // (only those pages are seen).
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (a.ctx[b] > a.max_pages * a.sub * 16 && threadIdx.x == 0) set_error(kErrShape);
    if (a.ctx[b] <= 0 || a.max_pages == 0)
      for (int i = threadIdx.x; i < a.heads * HD; i += D4_WARPS * 32) a.out[b * a.out_stride + i] = f2bf(0.f);
  }

  const int total = d4_total(a);
  const int runs = (int)gridDim.x * D4_WARPS;
  const int per = max(a.min_run, (total + runs - 1) / runs);
  // consecutive runs go to different SMs: few runs use all of them
  const int run = warp * (int)gridDim.x + (int)blockIdx.x;
  const int first = (int)min((int64_t)total, (int64_t)run * per), last = min(total, first + per);
  if (first >= last) return;
  if (lane == 0) {
    for (int i = 0; i < a.stages; ++i) mbar_init(&full[i], 2);
    fence_barrier_init();
  }
  __syncwarp();

  D4Cursor w = d4_at(a, first);
  // The ring's source: lane 2 i + r holds record r of the run's piece 16 k + i, k
  // growing, and copies it; the page ids of the next 16 pieces are on their way
  // meanwhile.
  D4Cursor ahead = w;
  ahead.advance(a, lane >> 1);
  auto look_up = [&]() {
    cp_async4(&pages[lane],
              a.tables + (size_t)ahead.b * a.max_pages + min((2 * ahead.c + (lane & 1)) / a.sub, a.max_pages - 1));
    cp_async_commit();
  };
  const uint8_t* src = nullptr;               // null: past the end of its sequence
  auto resolve = [&]() {                      // the looked-up records' addresses, then the next look-up
    cp_async_wait<0>();
    const int rec = 2 * ahead.c + (lane & 1);
    int page = pages[lane];
    src = nullptr;
    if (rec * 16 < ahead.len) {
      if ((unsigned)page >= (unsigned)a.num_pages) {               // read another page instead, and say so
        if (ahead.n != 0x7fffffff) set_error(kErrShape);
        page = 0;
      }
      src = a.cache + (((size_t)page * a.kv_heads + ahead.h) * a.sub + rec % a.sub) * REC;
    }
    ahead.advance(a, 16);
    look_up();
  };
  look_up();
  int issued = first, fill = 0;               // next piece of the run to fetch, its stage
  auto fetch = [&]() {
    const int k = (issued - first) & 15;
    if (k == 0) resolve();
    if ((lane >> 1) == k) {
      if (src != nullptr) {
        mbar_arrive_expect_tx(&full[fill], REC);
        bulk_load_1d(ring + (2 * fill + (lane & 1)) * REC, src, REC, &full[fill]);
      } else {
        mbar_arrive(&full[fill]);
      }
    }
    ++issued;
    if (++fill == a.stages) fill = 0;
  };
  for (int i = 0; i < a.stages && issued < last; ++i) fetch();

  Warp acc;
  acc.rs = rs[warp];
  int st = 0;
  uint32_t phase = 0;
  bool ok = true;                             // no wait has given up
  for (int at = first; at < last;) {
    const int c0 = w.c, c1 = min(w.n, c0 + (last - at));
    const __nv_bfloat16* q = a.q + w.b * a.q_stride + (int64_t)w.h * a.group * HD;
    acc.begin([&](int col) { return col < a.group ? q + col * HD : (const __nv_bfloat16*)nullptr; }, a.scale_log2);
    for (int c = c0; c < c1 && ok; ++c) {
      ok = __all_sync(0xffffffffu, kv4_wait(&full[st], phase, kErrD4Full));
      if (!ok) {
        // The copies under way land before the CTA gives its memory back.
        for (int left = issued - at - (c - c0); left > 0; --left) {
          kv4_drain(&full[st], phase);
          if (++st == a.stages) {
            st = 0;
            phase ^= 1u;
          }
        }
        break;
      }
      acc.tokens(ring + st * (2 * REC), w.len - c * 32);
      __syncwarp();
      if (issued < last) fetch();
      if (++st == a.stages) {
        st = 0;
        phase ^= 1u;
      }
    }
    // After a wait that gave up every segment of the run still arrives at its
    // joins, as NaN: the counters return to zero and no later call waits for it.
    if (!ok) acc.poison();
    acc.finish();
    __nv_bfloat16* out = a.out + w.b * a.out_stride + (int64_t)w.h * a.group * HD;
    bool done = c0 == 0 && c1 == w.n;
    if (!done) {
      // The runs of this segment, f to z, and the tree over them. A run has at
      // most two pieces of split segments: one that it does not begin (slot 0)
      // and one that it begins (slot 1).
      const int start = at - c0, f = start / per, z = (start + w.n - 1) / per;
      auto slot = [&](int r) { return 2 * r + (r == f); };
      acc.save(a.part + (size_t)slot(run) * Warp::PART);
      int lo = f, hi = z, x = run;           // the level's nodes of this segment, and ours
      for (int level = 0;; ++level) {
        const int g0 = max(lo, x & ~7), g1 = min(hi, x | 7);        // our group of eight
        auto left = [&](int y) { return max(f, y << (3 * level)); };   // a node's data lies with its leftmost run
        if (g1 > g0) {
          __syncwarp();                      // lane 0 releases every lane's part
          int old = 0;
          int* count = a.arrived + level * 2 * runs + slot(left(g0));
          if (lane == 0) old = atom_add_acq_rel(count, 1);
          __syncwarp();                      // and acquires the others' for every lane
          old = __shfl_sync(0xffffffffu, old, 0);
          if (old != g1 - g0) break;
          if (lane == 0) *count = 0;
          acc.join(g1 - g0 + 1, [&](int y) { return a.part + (size_t)slot(left(g0 + y)) * Warp::PART; });
          done = g0 == lo && g1 == hi;
          if (done) break;
          acc.save(a.part + (size_t)slot(left(g0)) * Warp::PART);
        }
        x >>= 3;
        lo >>= 3;
        hi >>= 3;
      }
    }
    if (done) {
      if (a.out_vec) acc.template store<true>(out, a.group);
      else acc.template store<false>(out, a.group);
    }
    at += c1 - c0;
    if (at < last) w.advance(a, c1 - c0);
  }
  cp_async_wait<0>();
}

template <int NG, int NH, int MIN_CTAS>
static void decode4_launch(Decode4Args a, int sms, cudaStream_t stream) {
  constexpr int STAGE = 4 * kv4_record(NG);
  constexpr int ROOM = 227 * 1024 / MIN_CTAS - 1024 - D4_WARPS * (D4_MAX_STAGES * 8 + D4_PAGES * 4 + NG * 4);
  a.stages = std::min(D4_MAX_STAGES, ROOM / (D4_WARPS * STAGE));
  const int smem = D4_WARPS * a.stages * STAGE;
  static const cudaError_t attr =
      cudaFuncSetAttribute(decode4_kernel<NG, NH, MIN_CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, ROOM);
  C10_CUDA_CHECK(attr);
  const int64_t most = (int64_t)a.batch * a.kv_heads * ((a.max_pages * a.sub + 1) / 2);
  const int grid = (int)std::min<int64_t>(sms * MIN_CTAS, std::max<int64_t>(1, most));
  constexpr int64_t RUN_BYTES = 2 * Kv4Warp<NG, NH>::PART * 16;
  TORCH_CHECK(grid * D4_WARPS * RUN_BYTES <= WS_PARTS && grid * D4_WARPS <= D4_MAX_RUNS,
              "paged_decode4: workspace too small for this GPU");
  decode4_kernel<NG, NH, MIN_CTAS><<<grid, D4_WARPS * 32, smem, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace dsv

// ---------------------------------------------------------------- bindings

int64_t dsv_kv4_workspace_bytes() { return dsv::WS_PARTS + dsv::D4_LEVELS * 2 * dsv::D4_MAX_RUNS * 4; }

// Returns the number of kernels launched.
int64_t dsv_paged_decode4(torch::Tensor q, torch::Tensor cache, torch::Tensor tables, torch::Tensor ctx,
                          torch::Tensor out, int64_t heads, double scale, torch::Tensor ws) {
  using namespace dsv;
  const int ng = dsv_kv4_groups(cache, "paged_decode4");
  const int64_t B = q.size(0), hkv = cache.size(1);
  TORCH_CHECK_VALUE(heads > 0 && heads % hkv == 0 && heads / hkv <= 16,
                    "paged_decode4: query heads must be 1 to 16 times the kv heads");
  TORCH_CHECK_VALUE(scale > 0, "paged_decode4: scale must be positive");
  for (const auto* x : {&q, &out})
    TORCH_CHECK_VALUE(x->is_cuda() && x->device() == cache.device() && x->scalar_type() == at::kBFloat16 &&
                          x->dim() == 2 && x->size(0) == B && x->size(1) == heads * HD && x->stride(1) == 1,
                      "paged_decode4: q and out must be bf16 [batch, heads * 128] with contiguous rows on the cache's device");
  TORCH_CHECK_VALUE(q.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
                    "paged_decode4: q rows must be 16-byte aligned");
  TORCH_CHECK_VALUE(tables.scalar_type() == at::kInt && tables.dim() == 2 && tables.size(0) == B && tables.is_contiguous() &&
                        ctx.scalar_type() == at::kInt && ctx.dim() == 1 && ctx.size(0) == B && ctx.is_contiguous() &&
                        tables.device() == cache.device() && ctx.device() == cache.device(),
                    "paged_decode4: block tables must be int32 [batch, pages], context lengths int32 [batch]");
  const int64_t most = tables.size(1) * cache.size(2) * 16;     // longest context
  TORCH_CHECK_VALUE(most < (int64_t(1) << 31) && B * hkv * (most / 32 + 1) < (int64_t(1) << 31),
                    "paged_decode4: block tables of more than 2^31 tokens");
  TORCH_CHECK_VALUE(ws.is_cuda() && ws.device() == cache.device() && ws.is_contiguous() &&
                        (int64_t)ws.nbytes() >= dsv_kv4_workspace_bytes(),
                    "paged_decode4: the workspace must come from kv4_workspace on the cache's device");
  if (B == 0) return 0;
  c10::cuda::CUDAGuard guard(cache.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  Decode4Args a{};
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.q_stride = q.stride(0);
  a.cache = cache.data_ptr<uint8_t>();
  a.tables = tables.data_ptr<int>();
  a.ctx = ctx.data_ptr<int>();
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.out_stride = out.stride(0);
  a.out_vec = out.stride(0) % 2 == 0 && reinterpret_cast<uintptr_t>(out.data_ptr()) % 4 == 0;
  a.part = reinterpret_cast<float4*>(ws.data_ptr());
  a.arrived = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(ws.data_ptr()) + WS_PARTS);
  a.batch = (int)B;
  a.max_pages = (int)tables.size(1);
  a.num_pages = (int)cache.size(0);
  a.heads = (int)heads;
  a.kv_heads = (int)hkv;
  a.group = (int)(heads / hkv);
  a.sub = (int)cache.size(2);
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.min_run = 2;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  if (a.group <= 8)
    ng == 1 ? decode4_launch<1, 1, 4>(a, sms, stream)
    : ng == 2 ? decode4_launch<2, 1, 4>(a, sms, stream) : decode4_launch<4, 1, 4>(a, sms, stream);
  else
    ng == 1 ? decode4_launch<1, 2, 2>(a, sms, stream)
    : ng == 2 ? decode4_launch<2, 2, 2>(a, sms, stream) : decode4_launch<4, 2, 2>(a, sms, stream);
  return 1;
}

DSV_ERROR_ACCESSOR(dsv_read_error_kv4_decode)
