// Verification of drafted tokens against the target's probabilities.
//
// Draft j of a request, token x, stays while u_j q_j[x] < p_j[x] (q = 1 where the
// drafts were certain), which keeps it with probability min(1, p / q). At the first
// refusal m the token is drawn from r = max(p_m - q_m, 0) instead, after m = all
// drafts from p_m: the smallest i with r_0 + .. + r_i > u_last * sum(r). The
// products and sums are f64: a float's 24 bits would decide borders by rounding
// (the products of two floats are exact in f64, and the order of a sum moves it
// by parts in 10^16).
//
// Bound by memory: of K + 1 rows only the two at m are read. One request's rows
// are 1 MB, so they are split over workgroups: k_verify_sums adds up one chunk of
// kVerifyChunk entries each (a later kernel rather than a counter joins them: no
// state to clear, and the sums' order never changes), k_verify_pick finds the
// chunk by the chunk sums and reads that chunk again, in order.
#include <hip/hip_runtime.h>

#include "ogkm/elem.hpp"
#include "ogkm/kernels.hpp"
#include "ogkm/paged.hpp"

namespace ogkm {

template <typename T>
struct VerifyRow {
  uint32_t m, count;   // accepted drafts, drafts
  const T* p;          // the target's row at m
  const T* q;          // the draft's row at m (null: none, or a certain draft)
  int32_t certain;     // the refused token of a certain draft, else -1
};

// Every wave finds m by itself: lane j tests draft j.
template <typename T>
__device__ __forceinline__ VerifyRow<T> verify_row(const VerifyArgs& a, uint32_t b) {
  const uint32_t lane = threadIdx.x & 63;
  const T* p = reinterpret_cast<const T*>(a.p) + b * a.p_batch;
  const T* q = a.q ? reinterpret_cast<const T*>(a.q) + b * a.q_batch : nullptr;
  VerifyRow<T> r;
  r.count = a.counts ? (uint32_t)min(max(a.counts[b], 0), (int32_t)a.K) : a.K;
  r.m = r.count;
  for (uint32_t j0 = 0; j0 < r.count; j0 += 64) {
    const uint32_t j = j0 + lane;
    bool stays = true;
    if (j < r.count) {
      const int32_t x = a.tokens[(uint64_t)b * a.K + j];
      stays = x >= 0 && (uint32_t)x < a.V;
      if (stays) {
        const double qt = q ? (double)to_f32<T>(q[j * a.q_row + x]) : 1.0;
        stays = (double)a.u[(uint64_t)b * a.K + j] * qt < (double)to_f32<T>(p[j * a.p_row + x]);
      }
    }
    const uint64_t gone = __ballot(!stays);
    if (gone) {
      r.m = j0 + (uint32_t)__builtin_ctzll(gone);
      break;
    }
  }
  r.p = p + r.m * a.p_row;
  r.q = q && r.m < r.count ? q + r.m * a.q_row : nullptr;
  r.certain = !q && r.m < r.count ? a.tokens[(uint64_t)b * a.K + r.m] : -1;
  return r;
}

// Weight of entry i in the residual; a NaN in either row weighs nothing.
__device__ __forceinline__ double residual(float p, float q) {
  return p > q && p > 0.f ? (double)p - (double)fmaxf(q, 0.f) : 0.0;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) k_verify_sums(VerifyArgs a) {
  __shared__ double part[4][2];
  const uint32_t b = blockIdx.y, tid = threadIdx.x;
  const VerifyRow<T> r = verify_row<T>(a, b);
  const uint32_t c0 = blockIdx.x * kVerifyChunk;
  double res = 0.0, all = 0.0;
#pragma unroll
  for (uint32_t k = 0; k < kVerifyChunk / 256; ++k) {
    const uint32_t i = c0 + k * 256 + tid;
    if (i < a.V) {
      const float p = to_f32<T>(r.p[i]);
      const float q = r.q ? to_f32<T>(r.q[i]) : (int32_t)i == r.certain ? 1.f : 0.f;
      res += residual(p, q);
      all += p > 0.f ? (double)p : 0.0;
    }
  }
  res = wave_sum_f64(res);
  all = wave_sum_f64(all);
  if ((tid & 63) == 0) {
    part[tid >> 6][0] = res;
    part[tid >> 6][1] = all;
  }
  __syncthreads();
  if (tid < 2)
    a.sums[((uint64_t)b * gridDim.x + blockIdx.x) * 2 + tid] = part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid];
}

template <typename T>
__global__ void __launch_bounds__(256) k_verify_pick(VerifyArgs a) {
  __shared__ double part[4];
  __shared__ int32_t pick_s, last_s;
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t nchunks = (a.V + kVerifyChunk - 1) / kVerifyChunk;
  const VerifyRow<T> r = verify_row<T>(a, b);
  const double* sums = a.sums + (uint64_t)b * nchunks * 2;
  // totals, then the chunk: every wave for itself, in the same order
  double res = 0.0, all = 0.0;
  for (uint32_t c = lane; c < nchunks; c += 64) {
    res += sums[2 * c];
    all += sums[2 * c + 1];
  }
  res = wave_sum_f64(res);
  all = wave_sum_f64(all);
  const bool use_res = res > 0.0;
  const double aim = (double)a.u_last[b] * (use_res ? res : all);
  double before = 0.0, chunk_before = 0.0;
  int32_t chunk = -1;   // first chunk whose running sum passes the aim, else the last with any weight
  bool found = false;
  for (uint32_t c0 = 0; c0 < nchunks && !found; c0 += 64) {
    const double own = c0 + lane < nchunks ? sums[2 * (c0 + lane) + (use_res ? 0 : 1)] : 0.0;
    double x = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(x, o, 64);
      if ((int)lane >= o) x += y;
    }
    const double to = before + x;
    const uint64_t past = __ballot(own > 0.0 && to > aim), some = __ballot(own > 0.0);
    found = past != 0;
    if (past || some) {
      const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
      chunk = (int32_t)c0 + l;
      chunk_before = __shfl(to - own, l, 64);
    }
    before = __shfl(to, 63, 64);
  }
  if (tid == 0) {
    pick_s = INT32_MAX;
    last_s = -1;
  }
  __syncthreads();
  if (chunk >= 0) {
    constexpr uint32_t kOwn = kVerifyChunk / 256;  // consecutive entries of a thread
    const uint32_t i0 = (uint32_t)chunk * kVerifyChunk + tid * kOwn;
    double w[kOwn], mine = 0.0;
#pragma unroll
    for (uint32_t k = 0; k < kOwn; ++k) {
      const uint32_t i = i0 + k;
      w[k] = 0.0;
      if (i < a.V) {
        const float p = to_f32<T>(r.p[i]);
        const float q = !use_res ? 0.f : r.q ? to_f32<T>(r.q[i]) : (int32_t)i == r.certain ? 1.f : 0.f;
        w[k] = residual(p, q);
      }
      mine += w[k];
    }
    double x = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(x, o, 64);
      if ((int)lane >= o) x += y;
    }
    if (lane == 63) part[wave] = x;
    __syncthreads();
    double c = chunk_before + x - mine;
    for (uint32_t v = 0; v < wave; ++v) c += part[v];
    int32_t pick = INT32_MAX, last = -1;
#pragma unroll
    for (uint32_t k = 0; k < kOwn; ++k) {
      c += w[k];
      if (w[k] > 0.0) {
        last = (int32_t)(i0 + k);
        if (c > aim && pick == INT32_MAX) pick = last;
      }
    }
    if (pick != INT32_MAX) atomicMin(&pick_s, pick);  // LDS, integers: the order does not matter
    if (last >= 0) atomicMax(&last_s, last);
    __syncthreads();
  }
  const int32_t token = pick_s != INT32_MAX ? pick_s : last_s;
  for (uint32_t j = tid; j <= a.K; j += 256)
    a.out[(uint64_t)b * (a.K + 1) + j] = j < r.m ? a.tokens[(uint64_t)b * a.K + j] : j == r.m ? token : -1;
  if (tid == 0) a.accepted[b] = (int32_t)r.m;
}

hipError_t launch_verify_draft(const VerifyArgs& a, hipStream_t s) {
  if (!a.V || a.B > 65535) return hipErrorInvalidValue;
  if (!a.B) return hipSuccess;
  const dim3 grid((a.V + kVerifyChunk - 1) / kVerifyChunk, a.B);
#define OGKM_VERIFY(T)                                                          \
  do {                                                                          \
    hipLaunchKernelGGL((k_verify_sums<T>), grid, dim3(256), 0, s, a);           \
    hipLaunchKernelGGL((k_verify_pick<T>), dim3(a.B), dim3(256), 0, s, a);      \
  } while (0)
  if (a.elem == ELEM_F32)
    OGKM_VERIFY(float);
  else if (a.elem == ELEM_F16)
    OGKM_VERIFY(_Float16);
  else
    OGKM_VERIFY(__bf16);
#undef OGKM_VERIFY
  return hipGetLastError();
}

}  // namespace ogkm
