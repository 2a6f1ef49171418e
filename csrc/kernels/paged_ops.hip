// The step around paged attention (csrc/kernels/paged_attn.hip):
//   k_plan        where every new token of a batch goes: pages handed out of the
//                 free list, block-table rows extended, positions and slots
//   k_paged_rope  rotate-half RoPE of q and k at one position per row, k and v
//                 stored into their slots of the page pool
#include <hip/hip_runtime.h>

#include "ogkm/elem.hpp"
#include "ogkm/kernels.hpp"
#include "ogkm/paged.hpp"

namespace ogkm {

// ---------------------------------------------------------------- step plan
// Two prefix sums over the requests (rows, then pages needed) decide everything:
//   end_b   = sum of new_lens up to b              (rows of b: [end_b - new_b, end_b))
//   need_b  = max(0, ceil((kv_b + new_b) / P) - held_b)
//   upto_b  = sum of need up to b                  (free-list entries of b: [upto_b - need_b, upto_b))
//   granted = the pages fit the table row and the free list, the rows fit n_tokens
//             (a refused request's pages stay in upto: those behind it that lack
//             pages are refused too and cannot overtake it; prefix sums do not
//             depend on what was granted, a first-fit rule would be sequential)
// The op moves a few KB: its time is one launch and a chain of four dependent
// memory rounds (lengths -> scan -> table or free list -> store). So it is ONE
// launch: every workgroup scans all requests by itself (LDS keeps 9 bytes of
// each) rather than waiting for another's result, then takes its share of the
// new pages and of the token rows, finding a row's request by binary search.
// A token's page is read from the table only where the request held it before;
// new pages come from the free list directly, so no workgroup reads what
// another writes.
// A thread takes one request and one row where it can (1024 threads a workgroup;
// 256 for the few requests of a decode step): four of each in turn made it 12.2
// us instead of 8.4 for 1024 requests with 25000 rows.

// Exclusive prefix sum over the workgroup's threads; `total` is everyone's sum.
template <uint32_t NT>
__device__ __forceinline__ int64_t block_exclusive(int64_t v, int64_t* wave_sums, int64_t* total) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, 64);
    if ((int)lane >= o) x += y;
  }
  __syncthreads();  // wave_sums of an earlier call may still be read
  if (lane == 63) wave_sums[wave] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < NT / 64; ++w) {
    if (w < wave) before += wave_sums[w];
    all += wave_sums[w];
  }
  *total = all;
  return before + x - v;
}

// First index i of [0, n) with a[i + 1] > x (a ascending, a[0] <= x < a[n]).
__device__ __forceinline__ uint32_t owner_of(const int32_t* a, uint32_t n, int32_t x) {
  uint32_t lo = 0, hi = n - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) >> 1;
    if (a[mid + 1] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

template <uint32_t NT>
__global__ void __launch_bounds__(NT) k_plan(PlanArgs a) {
  extern __shared__ int32_t plan_lds[];
  int32_t* cu = plan_lds;             // [B + 1] first row of each request
  int32_t* up = plan_lds + a.B + 1;   // [B + 1] first new page of each request
  uint8_t* ok = reinterpret_cast<uint8_t*>(plan_lds + 2 * (a.B + 1));
  __shared__ int64_t wave_sums[NT / 64];
  __shared__ int32_t taken_s;
  const uint32_t tid = threadIdx.x;
  const uint32_t per = (a.B + NT - 1) / NT;
  const uint32_t b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  const int64_t round = (1ll << a.page_shift) - 1;
  const int32_t raw_start = a.free_start[0];
  const int64_t start = min((int64_t)max(raw_start, 0), (int64_t)a.n_free);
  if (tid == 0) {
    cu[0] = up[0] = 0;
    taken_s = 0;
  }
  int64_t rows = 0, total;
  for (uint32_t b = b0; b < b1; ++b) rows += max(a.new_lens[b], 0);
  int64_t end = block_exclusive<NT>(rows, wave_sums, &total);
  int64_t pages = 0;
  for (uint32_t b = b0; b < b1; ++b) {
    const int64_t fresh = max(a.new_lens[b], 0), kv = max(a.kv_lens[b], 0);
    const int64_t have = min((int64_t)max(a.page_counts[b], 0), (int64_t)a.width);
    end += fresh;
    cu[b + 1] = (int32_t)min(end, (int64_t)a.n_tokens);
    const int64_t held = (kv + fresh + round) >> a.page_shift;
    const bool fits = held <= (int64_t)a.width && end <= (int64_t)a.n_tokens;
    const int64_t need = fits ? max(held - have, (int64_t)0) : 0;
    ok[b] = fits;
    up[b + 1] = (int32_t)need;  // at most the width; summed below
    pages += need;
  }
  int64_t upto = block_exclusive<NT>(pages, wave_sums, &total);
  int32_t taken = 0;
  for (uint32_t b = b0; b < b1; ++b) {
    const int32_t need = up[b + 1];
    upto += need;
    const bool granted = ok[b] && (need == 0 || start + upto <= (int64_t)a.n_free);
    ok[b] = granted;
    up[b + 1] = (int32_t)min(upto, (int64_t)INT32_MAX);
    if (granted && need) taken = (int32_t)upto;  // grants of pages are a prefix: upto only grows
    if (blockIdx.x == 0) {
      const int32_t kv = max(a.kv_lens[b], 0), fresh = max(a.new_lens[b], 0);
      const int32_t have = min(max(a.page_counts[b], 0), (int32_t)a.width);
      a.cu_q[b + 1] = cu[b + 1];
      a.kv_out[b] = granted ? kv + fresh : kv;
      a.counts_out[b] = have + (granted ? need : 0);
      a.granted[b] = granted;
    }
  }
  if (taken) atomicMax(&taken_s, taken);  // LDS, integers: the order does not matter
  __syncthreads();
  taken = taken_s;
  if (blockIdx.x == 0 && tid == 0) {
    a.cu_q[0] = 0;
    a.free_out[0] = (int32_t)(start + taken);
  }
  const uint32_t stride = gridDim.x * NT, first = blockIdx.x * NT + tid;
  for (uint32_t p = first; p < (uint32_t)taken; p += stride) {
    const uint32_t b = owner_of(up, a.B, (int32_t)p);
    const int32_t have = min(max(a.page_counts[b], 0), (int32_t)a.width);
    a.table[b * a.table_ld + have + (p - up[b])] = a.free_pages[start + p];
  }
  const int32_t rows_all = a.B ? cu[a.B] : 0;
  for (uint32_t t = first; t < a.n_tokens; t += stride) {
    int32_t pos = -1, slot = -1;
    if ((int32_t)t < rows_all) {
      const uint32_t b = owner_of(cu, a.B, (int32_t)t);
      if (ok[b]) {
        pos = max(a.kv_lens[b], 0) + (int32_t)(t - cu[b]);
        const int32_t have = min(max(a.page_counts[b], 0), (int32_t)a.width);
        const int32_t at = pos >> a.page_shift;
        const int32_t page = at < have ? a.table[b * a.table_ld + at] : a.free_pages[start + up[b] + (at - have)];
        if (page >= 0 && page <= (INT32_MAX >> a.page_shift))
          slot = (page << a.page_shift) + (pos & (int32_t)round);
      }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
}

hipError_t launch_paged_plan(const PlanArgs& a, hipStream_t s) {
  if (a.B > kPlanMaxRequests || a.page_shift > 16) return hipErrorInvalidValue;
  const uint32_t threads = a.B <= 256 && a.n_tokens <= 256 ? 256 : 1024;
  const uint32_t grid = min(max((a.n_tokens + threads - 1) / threads, 1u), 1024u);
  const size_t lds = (size_t)(a.B + 1) * 8 + a.B;
  if (threads == 256)
    hipLaunchKernelGGL((k_plan<256>), dim3(grid), dim3(threads), lds, s, a);
  else
    hipLaunchKernelGGL((k_plan<1024>), dim3(grid), dim3(threads), lds, s, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------- RoPE into pages
// Bound by memory: each element of qkv is read once and written once. A thread
// takes 8 pairs (i, i + hd / 2) of one head of one row: two 16-byte loads, two
// 16-byte stores. cos and sin rows are shared by all heads of a row and come
// from the caches. Math in f32, one rounding to the element type.
template <typename T>
__global__ void __launch_bounds__(256) k_paged_rope(PagedRopeArgs a) {
  typedef typename Vec<T>::v8 v8;
  const uint32_t half = a.hd / 2, chunks = half / 8, heads = a.hq + 2 * a.hkv;
  const uint32_t per_row = heads * chunks;
  const uint32_t item = blockIdx.x * 256 + threadIdx.x;  // the launcher keeps items below 2^32
  const uint32_t t = item / per_row;
  if (t >= a.n) return;
  const uint32_t rest = item - t * per_row, h = rest / chunks, i = (rest - h * chunks) * 8;
  const int32_t pos = a.positions[t], slot = a.slots[t];
  const uint16_t* src = a.qkv + t * a.ldqkv + (uint64_t)h * a.hd + i;
  v8 x1 = *reinterpret_cast<const v8*>(src), x2 = *reinterpret_cast<const v8*>(src + half);
  if (h < a.hq + a.hkv) {
    if (pos < 0) {  // a padding row
      x1 = x2 = v8{};
    } else {
      const bool in = (uint32_t)pos < a.max_pos;
      const float* c = a.cos + (uint64_t)(in ? pos : 0) * half + i;
      const float* s = a.sin + (uint64_t)(in ? pos : 0) * half + i;
      float cv[8], sv[8];
      *reinterpret_cast<f32x4_t*>(cv) = *reinterpret_cast<const f32x4_t*>(c);
      *reinterpret_cast<f32x4_t*>(cv + 4) = *reinterpret_cast<const f32x4_t*>(c + 4);
      *reinterpret_cast<f32x4_t*>(sv) = *reinterpret_cast<const f32x4_t*>(s);
      *reinterpret_cast<f32x4_t*>(sv + 4) = *reinterpret_cast<const f32x4_t*>(s + 4);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float u = to_f32<T>(x1[j]), v = to_f32<T>(x2[j]);
        const float cj = in ? cv[j] : __builtin_nanf(""), sj = sv[j];
        x1[j] = from_f32<T>(u * cj - v * sj);
        x2[j] = from_f32<T>(v * cj + u * sj);
      }
    }
  }
  uint16_t* dst;
  if (h < a.hq) {
    dst = a.q_out + ((uint64_t)t * a.hq + h) * a.hd;
  } else {
    const uint32_t page = (uint32_t)slot >> a.page_shift;
    if (pos < 0 || slot < 0 || page >= a.num_pages) return;
    const uint32_t kv = h < a.hq + a.hkv ? 0u : 1u;
    dst = a.pages + kv * a.kv_stride + page * a.page_stride + (h - a.hq - kv * a.hkv) * a.head_stride +
          (uint64_t)((uint32_t)slot & ((1u << a.page_shift) - 1u)) * a.hd;
  }
  *reinterpret_cast<v8*>(dst + i) = x1;
  *reinterpret_cast<v8*>(dst + i + half) = x2;
}

hipError_t launch_paged_rope(const PagedRopeArgs& a, hipStream_t s) {
  if (a.hd % 16 || !a.hd || a.page_shift > 16) return hipErrorInvalidValue;
  const uint64_t items = (uint64_t)a.n * (a.hq + 2 * a.hkv) * (a.hd / 16);
  if (items + 255 > UINT32_MAX) return hipErrorInvalidValue;
  if (!items) return hipSuccess;
  const dim3 grid((uint32_t)((items + 255) / 256));
  if (a.elem == ELEM_F16)
    hipLaunchKernelGGL((k_paged_rope<_Float16>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((k_paged_rope<__bf16>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace ogkm
