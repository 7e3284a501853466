// Decode attention over the 4-bit paged KV cache (format and tile arithmetic:
// kv4.cuh): one query token per sequence, grouped heads, fp32 softmax.
//
// The reference project decodes over its serving library's bf16 pages; this is
// the same function over the values the codes stand for.
//
// One CTA = (context split, KV head, sequence), four warps; a warp takes every
// fourth 16-token record of the split and keeps its own softmax state, so the
// loop has no barrier. The GQA group's query heads are the columns of the warp's
// matrix tiles and share every byte read. Splits of one (sequence, head) leave
// (max, sum, output) partials in the workspace for a second kernel.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "kv4.cuh"

int dsv_kv4_groups(const torch::Tensor& cache, const char* op);

namespace dsv {

constexpr int D4_WARPS = 4;

struct Decode4Args {
  const __nv_bfloat16* q;   // [B, Hq * 128], row stride q_stride
  int64_t q_stride;
  const uint8_t* cache;
  const int* tables;        // [B, max_pages]
  const int* ctx;           // [B]
  __nv_bfloat16* out;       // [B, Hq * 128], row stride out_stride
  int64_t out_stride;
  float* part;              // [B, Hq, splits, 130]
  int max_pages, num_pages, heads, kv_heads, group, sub, splits;   // sub: records per page
  float scale_log2;
};

template <int NG, int NH>
__global__ void __launch_bounds__(D4_WARPS * 32) decode4_kernel(Decode4Args a) {
  __shared__ float so[D4_WARPS][NH * 8][HD + 4];
  __shared__ float sm[D4_WARPS][NH * 8], sl[D4_WARPS][NH * 8];
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ctx = min(a.ctx[b], a.max_pages * a.sub * 16);
  const int recs = (ctx + 15) / 16, per = (recs + a.splits - 1) / a.splits;
  const int r0 = split * per, r1 = min(recs, r0 + per);
  const int* tab = a.tables + (size_t)b * a.max_pages;
  Kv4Warp<NG, NH> w;
  const __nv_bfloat16* q = a.q + b * a.q_stride + (int64_t)kvh * a.group * HD;
  w.begin([&](int c) { return c < a.group ? q + c * HD : (const __nv_bfloat16*)nullptr; }, a.scale_log2);
  for (int r = r0 + warp; r < r1; r += D4_WARPS) {
    const int page = tab[r / a.sub];
    if ((unsigned)page >= (unsigned)a.num_pages) {
      if (lane == 0) set_error(kErrShape);
      continue;
    }
    const uint8_t* rec = a.cache + (((size_t)page * a.kv_heads + kvh) * a.sub + r % a.sub) * (2 * kv4_record(NG));
    const int valid = ctx - r * 16;
    w.tile(rec, [&](int tok, int) { return tok < valid; });
  }
  w.finish();
#pragma unroll
  for (int n = 0; n < NH; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int col = n * 8 + 2 * t + c;
      if (g == 0) {
        sm[warp][col] = w.m[n][c];
        sl[warp][col] = w.l[n][c];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        so[warp][col][16 * i + g] = w.out(n, i, c);
        so[warp][col][16 * i + g + 8] = w.out(n, i, 2 + c);
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < a.group * HD; i += D4_WARPS * 32) {
    const int c = i / HD, d = i % HD;
    float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
    for (int x = 0; x < D4_WARPS; ++x) M = fmaxf(M, sm[x][c]);
#pragma unroll
    for (int x = 0; x < D4_WARPS; ++x) {
      if (sl[x][c] == 0.f) continue;   // no token seen (a NaN sum goes on)
      const float e = kv4_exp2(sm[x][c] - M);
      L += sl[x][c] * e;
      O += so[x][c][d] * e;
    }
    const int h = kvh * a.group + c;
    if (a.splits == 1) {
      a.out[b * a.out_stride + h * HD + d] = f2bf(L != 0.f ? O / L : 0.f);
    } else {
      float* p = a.part + (((size_t)b * a.heads + h) * a.splits + split) * (HD + 2);
      p[2 + d] = O;
      if (d == 0) {
        p[0] = M;
        p[1] = L;
      }
    }
  }
}

__global__ void __launch_bounds__(HD) decode4_join_kernel(Decode4Args a) {
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const float* p = a.part + ((size_t)b * a.heads + h) * a.splits * (HD + 2);
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, p[s * (HD + 2)]);
  for (int s = 0; s < a.splits; ++s) {
    const float m = p[s * (HD + 2)];
    if (p[s * (HD + 2) + 1] == 0.f) continue;
    const float e = kv4_exp2(m - M);
    L += p[s * (HD + 2) + 1] * e;
    O += p[s * (HD + 2) + 2 + d] * e;
  }
  a.out[b * a.out_stride + h * HD + d] = f2bf(L != 0.f ? O / L : 0.f);
}

}  // namespace dsv

// ---------------------------------------------------------------- bindings

int64_t dsv_kv4_workspace_bytes() { return 32 << 20; }

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
  a.part = reinterpret_cast<float*>(ws.data_ptr());
  a.max_pages = (int)tables.size(1);
  a.num_pages = (int)cache.size(0);
  a.heads = (int)heads;
  a.kv_heads = (int)hkv;
  a.group = (int)(heads / hkv);
  a.sub = (int)cache.size(2);
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  // about four CTAs per SM, at least 64 tokens each
  const int64_t most = std::max<int64_t>(1, (int64_t)a.max_pages * a.sub / 4);
  a.splits = (int)std::max<int64_t>(1, std::min<int64_t>(592 / (B * hkv), most));
  const dim3 grid((unsigned)a.splits, (unsigned)hkv, (unsigned)B);
  auto launch = [&](auto kernel) { kernel<<<grid, D4_WARPS * 32, 0, stream>>>(a); };
  if (a.group <= 8)
    ng == 1 ? launch(decode4_kernel<1, 1>) : ng == 2 ? launch(decode4_kernel<2, 1>) : launch(decode4_kernel<4, 1>);
  else
    ng == 1 ? launch(decode4_kernel<1, 2>) : ng == 2 ? launch(decode4_kernel<2, 2>) : launch(decode4_kernel<4, 2>);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (a.splits == 1) return 1;
  decode4_join_kernel<<<dim3((unsigned)heads, (unsigned)B), HD, 0, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return 2;
}

DSV_ERROR_ACCESSOR(dsv_read_error_kv4_decode)
