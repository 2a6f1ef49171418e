// Attention of new tokens over a paged KV cache:
//   o_i = sum_{t <= pos_i} softmax_t(scale q_i . k_t) v_t,   pos_i = kv - n + i
// for row i of a request with n new rows and kv cached tokens (the new ones
// among them).
#include <hip/hip_runtime.h>

#include "ogkm/elem.hpp"
#include "ogkm/kernels.hpp"
#include "ogkm/paged.hpp"

namespace ogkm {

// One wave per (row, query head): a lane scores one of 64 keys at a time, then
// the wave adds the keys' value rows, two dims per lane. Running maximum and
// sum in f32.
template <typename T>
__global__ void __launch_bounds__(256) k_paged_attn(PagedAttnArgs a) {
  __shared__ float qs[4][128];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t item = blockIdx.x * 4 + wave;
  const uint32_t t = item / a.hq, h = item - t * a.hq;
  if (t >= a.n) return;
  uint32_t lo = 0, hi = a.B;
  while (lo < hi) {  // first request that ends behind row t
    const uint32_t mid = (lo + hi) >> 1;
    if (a.cu_q[mid + 1] > (int32_t)t)
      hi = mid;
    else
      lo = mid + 1;
  }
  if (lo == a.B || a.cu_q[lo] > (int32_t)t) return;
  const uint32_t b = lo;
  const int32_t n = min(a.cu_q[b + 1], (int32_t)a.n) - a.cu_q[b];
  const int32_t kv = max(a.kv_lens[b], 0);
  const int64_t pos = (int64_t)kv - n + ((int32_t)t - a.cu_q[b]);
  const uint64_t kvh = h / (a.hq / a.hkv);
  const T* q = reinterpret_cast<const T*>(a.q) + t * a.q_stride + h * a.q_head_stride;
  for (uint32_t d = lane; d < a.hd; d += 64) qs[wave][d] = to_f32<T>(q[d]) * a.scale;
  __builtin_amdgcn_wave_barrier();
  const int32_t* row = a.table + b * a.table_ld;
  const T* k0 = reinterpret_cast<const T*>(a.pages) + kvh * a.head_stride;
  const uint32_t mask = (1u << a.page_shift) - 1;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  bool bad = kv > ((int64_t)a.width << a.page_shift);
  for (int64_t base = 0; base <= pos && !bad; base += 64) {
    const int64_t key = base + lane;
    float sc = -INFINITY;
    uint64_t off = 0;
    bool miss = false;
    if (key <= pos) {
      const int32_t page = row[key >> a.page_shift];
      miss = page < 0 || (uint32_t)page >= a.num_pages;
      if (!miss) {
        off = page * a.page_stride + (key & mask) * a.hd;
        sc = 0.f;
        for (uint32_t d = 0; d < a.hd; ++d) sc += qs[wave][d] * to_f32<T>(k0[off + d]);
      }
    }
    bad = __any(miss);
    if (bad) break;
    float mx = sc;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const float mn = fmaxf(m, mx);
    const float f = m == -INFINITY ? 0.f : __expf(m - mn);
    const float p = key <= pos ? __expf(sc - mn) : 0.f;
    float ps = p;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ps += __shfl_xor(ps, o, 64);
    l = l * f + ps;
    o0 *= f;
    o1 *= f;
    m = mn;
    const int cnt = pos - base + 1 < 64 ? (int)(pos - base + 1) : 64;
    for (int j = 0; j < cnt; ++j) {
      const float pj = __shfl(p, j, 64);
      const uint64_t oj = __shfl(off, j, 64);
      const T* v = k0 + a.kv_stride + oj;
      if (2 * lane < a.hd) {
        o0 += pj * to_f32<T>(v[2 * lane]);
        o1 += pj * to_f32<T>(v[2 * lane + 1]);
      }
    }
  }
  if (2 * lane < a.hd) {
    T* out = reinterpret_cast<T*>(a.out) + t * a.out_stride + (uint64_t)h * a.hd + 2 * lane;
    const float none = bad ? __builtin_nanf("") : 0.f;
    out[0] = from_f32<T>(bad || pos < 0 ? none : o0 / l);
    out[1] = from_f32<T>(bad || pos < 0 ? none : o1 / l);
  }
}

hipError_t launch_paged_attn(const PagedAttnArgs& a, hipStream_t s) {
  if (!a.hkv || a.hq % a.hkv || (a.hd != 64 && a.hd != 128) || a.page_shift > 16) return hipErrorInvalidValue;
  const uint64_t waves = (uint64_t)a.n * a.hq;
  if (!waves || !a.B) return hipSuccess;
  const dim3 grid((uint32_t)((waves + 3) / 4));
  if (a.elem == ELEM_F16)
    hipLaunchKernelGGL((k_paged_attn<_Float16>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((k_paged_attn<__bf16>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace ogkm
