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
// Bound by memory: of K + 1 rows only the two at m are read, once; and, for few
// requests, by the chain of dependent reads. k_verify_sums finds m and adds up
// the residual of one chunk of kVerifyChunk entries a workgroup; k_verify_pick
// finds the chunk by the chunk sums, reads that chunk again, and scans it. A
// second launch joins the sums, not a counter: no state to clear, and the order
// of the sums never changes. (One launch with one workgroup a request was
// tried: the f64 sums of 128256 entries keep one CU busy for 30 us.)
#include <hip/hip_runtime.h>

#include "ogkm/elem.hpp"
#include "ogkm/kernels.hpp"
#include "ogkm/paged.hpp"

namespace ogkm {

template <typename T>
struct VerifyRow {
  uint32_t m;          // accepted drafts
  const T* p;          // the target's row at m
  const T* q;          // the draft's row at m (null: none, or a certain draft)
  int32_t certain;     // the refused token of a certain draft, else -1
};

// Every wave finds m by itself: lane j tests draft j. The lists are read
// before the count is known (K of them exist), one round of latency for all.
template <typename T>
__device__ __forceinline__ uint32_t accepted_drafts(const VerifyArgs& a, uint32_t b, uint32_t count) {
  const uint32_t lane = threadIdx.x & 63;
  const T* p = reinterpret_cast<const T*>(a.p) + b * a.p_batch;
  const T* q = a.q ? reinterpret_cast<const T*>(a.q) + b * a.q_batch : nullptr;
  for (uint32_t j0 = 0; j0 < a.K; j0 += 64) {
    const uint32_t j = j0 + lane;
    bool stays = true;
    if (j < a.K) {
      const int32_t x = a.tokens[(uint64_t)b * a.K + j];
      const double u = a.u[(uint64_t)b * a.K + j];
      stays = x >= 0 && (uint32_t)x < a.V;
      if (stays) {
        const double qt = q ? (double)to_f32<T>(q[j * a.q_row + x]) : 1.0;
        stays = u * qt < (double)to_f32<T>(p[j * a.p_row + x]);
      }
    }
    const uint64_t gone = __ballot(!stays);
    if (gone) return min(j0 + (uint32_t)__builtin_ctzll(gone), count);
    if (j0 + 64 >= count) return count;
  }
  return count;
}

__device__ __forceinline__ uint32_t draft_count(const VerifyArgs& a, uint32_t b) {
  return a.counts ? (uint32_t)min(max(a.counts[b], 0), (int32_t)a.K) : a.K;
}

template <typename T>
__device__ __forceinline__ VerifyRow<T> verify_row(const VerifyArgs& a, uint32_t b, uint32_t m, uint32_t count) {
  VerifyRow<T> r;
  r.m = m;
  r.p = reinterpret_cast<const T*>(a.p) + b * a.p_batch + m * a.p_row;
  r.q = a.q && m < count ? reinterpret_cast<const T*>(a.q) + b * a.q_batch + m * a.q_row : nullptr;
  r.certain = !a.q && m < count ? a.tokens[(uint64_t)b * a.K + m] : -1;
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

// Weights of entries i0 + k step (k < N) of a row, 0 behind its end; `whole`: of
// the target's row alone. All loads are issued before the first use (clamped
// indices, no branch around a load: one round of latency, not 2 N).
template <typename T, uint32_t N>
__device__ __forceinline__ void weights(const VerifyRow<T>& r, uint32_t i0, uint32_t step, uint32_t V, bool whole,
                                        double (&w)[N]) {
  const T* qr = r.q && !whole ? r.q : r.p;
  const bool no_q = whole || !r.q;
  T p[N], q[N];
  constexpr uint32_t E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(E), aligned(sizeof(T))));  // rows of an odd length begin anywhere
  if (step == 1 && i0 + N <= V) {
    // consecutive entries: 16 bytes a load, or the lanes' 64-byte stride costs a
    // cache line for each of them
#pragma unroll
    for (uint32_t k = 0; k < N; k += E) *reinterpret_cast<vec*>(p + k) = *reinterpret_cast<const vec*>(r.p + i0 + k);
#pragma unroll
    for (uint32_t k = 0; k < N; k += E) *reinterpret_cast<vec*>(q + k) = *reinterpret_cast<const vec*>(qr + i0 + k);
  } else {
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) p[k] = r.p[min(i0 + k * step, V - 1)];
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) q[k] = qr[min(i0 + k * step, V - 1)];
  }
#pragma unroll
  for (uint32_t k = 0; k < N; ++k) {
    const uint32_t i = i0 + k * step;
    const float qf = no_q ? (!whole && (int32_t)i == r.certain ? 1.f : 0.f) : to_f32<T>(q[k]);
    w[k] = i < V ? residual(to_f32<T>(p[k]), qf) : 0.0;
  }
}

// Sum of the calling wave's quarter of a chunk: 16 entries a lane, all loads in
// flight before the first use, 16 bytes each but in the row's last quarter.
template <typename T>
__device__ __forceinline__ double quarter_sum(const VerifyRow<T>& r, uint32_t i0, uint32_t V) {
  constexpr uint32_t E = 16 / sizeof(T), N = kVerifyChunk / 4 / 64 / E;  // entries of a load, loads
  typedef T vec __attribute__((ext_vector_type(E), aligned(sizeof(T))));
  const uint32_t lane = threadIdx.x & 63;
  double sum = 0.0;
  if (i0 + kVerifyChunk / 4 <= V) {
    vec p[N], q[N];
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) p[k] = *reinterpret_cast<const vec*>(r.p + i0 + (k * 64 + lane) * E);
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) q[k] = r.q ? *reinterpret_cast<const vec*>(r.q + i0 + (k * 64 + lane) * E) : vec{};
#pragma unroll
    for (uint32_t k = 0; k < N; ++k)
#pragma unroll
      for (uint32_t e = 0; e < E; ++e) {
        const bool is = (int32_t)(i0 + (k * 64 + lane) * E + e) == r.certain;
        sum += residual(to_f32<T>(p[k][e]), is ? 1.f : to_f32<T>(q[k][e]));
      }
  } else {
    double w[kVerifyChunk / 4 / 64];
    weights<T>(r, i0 + lane, 64, V, false, w);
#pragma unroll
    for (uint32_t k = 0; k < kVerifyChunk / 4 / 64; ++k) sum += w[k];
  }
  return wave_sum_f64(sum);
}

// Sum of this lane's value and the lower lanes'.
__device__ __forceinline__ double wave_scan_f64(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o, 64);
    if ((int)(threadIdx.x & 63) >= o) x += y;
  }
  return x;
}

template <typename T>
__global__ void __launch_bounds__(256) k_verify_sums(VerifyArgs a) {
  __shared__ double part[4];
  const uint32_t b = blockIdx.y, tid = threadIdx.x;
  const uint32_t count = draft_count(a, b), m = accepted_drafts<T>(a, b, count);
  const VerifyRow<T> r = verify_row<T>(a, b, m, count);
  const double sum = quarter_sum<T>(r, blockIdx.x * kVerifyChunk + (tid >> 6) * (kVerifyChunk / 4), a.V);
  if ((tid & 63) == 0) part[tid >> 6] = sum;
  __syncthreads();
  if (tid == 0) {
    a.sums[(uint64_t)b * gridDim.x + blockIdx.x] = part[0] + part[1] + part[2] + part[3];
    if (blockIdx.x == 0) a.accepted[b] = (int32_t)m;
  }
}

constexpr uint32_t kPickThreads = 256;

// One workgroup a request; its threads scan a chunk in order, 16 entries each.
// The code stays short on purpose (one instance of the scan): with a single
// workgroup the instructions come from L2 too.
template <typename T>
__global__ void __launch_bounds__(kPickThreads) k_verify_pick(VerifyArgs a) {
  constexpr uint32_t W = kPickThreads / 64, kOwn = kVerifyChunk / kPickThreads;
  __shared__ double part[W];
  __shared__ int32_t pick_s, last_s;
  const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t nchunks = (a.V + kVerifyChunk - 1) / kVerifyChunk;
  const double* sums = a.sums + (uint64_t)b * nchunks;
  const double u = a.u_last[b], sum0 = lane < nchunks ? sums[lane] : 0.0;
  const uint32_t m = (uint32_t)a.accepted[b];
  const VerifyRow<T> r = verify_row<T>(a, b, m, draft_count(a, b));
  if (tid == 0) {
    pick_s = INT32_MAX;
    last_s = -1;
  }
  const double upto0 = wave_scan_f64(sum0);
  double total = __shfl(upto0, 63, 64);
  if (nchunks > 64) {
    double rest = 0.0;
    for (uint32_t c = 64 + lane; c < nchunks; c += 64) rest += sums[c];
    total += wave_sum_f64(rest);
  }
  // Nothing remains of the target: its own row, walked by this workgroup alone,
  // once for the sum and once for the entry.
  const bool whole = !(total > 0.0);
  double aim = whole ? __builtin_inf() : u * total, before = 0.0;
  uint32_t c_begin = 0, c_end = nchunks;
  if (!whole) {
    // the first chunk whose running sum passes the aim, else the last with any
    // weight: every wave for itself, in the same order
    double run = 0.0;
    for (uint32_t c0 = 0; c0 < nchunks; c0 += 64) {
      const double own = c0 == 0 ? sum0 : c0 + lane < nchunks ? sums[c0 + lane] : 0.0;
      const double to = c0 == 0 ? upto0 : run + wave_scan_f64(own);
      const uint64_t past = __ballot(own > 0.0 && to > aim), some = __ballot(own > 0.0);
      if (some) {
        const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
        c_begin = c0 + l;
        before = __shfl(to - own, l, 64);
      }
      if (past) break;
      run = __shfl(to, 63, 64);
    }
    c_end = c_begin + 1;
  }
#pragma unroll 1
  for (int pass = whole ? 0 : 1; pass < 2; ++pass) {
#pragma unroll 1
    for (uint32_t c = c_begin; c < c_end; ++c) {
      const uint32_t i0 = c * kVerifyChunk + tid * kOwn;
      double w[kOwn], mine = 0.0;
      weights<T>(r, i0, 1, a.V, whole, w);
#pragma unroll
      for (uint32_t k = 0; k < kOwn; ++k) mine += w[k];
      const double x = wave_scan_f64(mine);
      __syncthreads();  // pick_s is set, and the chunk before is done with `part`
      if (lane == 63) part[wave] = x;
      __syncthreads();
      double run = before + x - mine;
#pragma unroll
      for (uint32_t v = 0; v < W; ++v) {
        if (v < wave) run += part[v];
        before += part[v];
      }
      int32_t pick = INT32_MAX, last = -1;
#pragma unroll
      for (uint32_t k = 0; k < kOwn; ++k) {
        run += w[k];
        if (w[k] > 0.0) {
          last = (int32_t)(i0 + k);
          if (run > aim && pick == INT32_MAX) pick = last;
        }
      }
      // lanes are in order: the wave's first pick, its last weight, one LDS atomic each
      const uint64_t picks = __ballot(pick != INT32_MAX), lasts = __ballot(last >= 0);
      if (picks && lane == (uint32_t)__builtin_ctzll(picks)) atomicMin(&pick_s, pick);
      if (lasts && lane == 63u - (uint32_t)__builtin_clzll(lasts)) atomicMax(&last_s, last);
      __syncthreads();
      if (pick_s != INT32_MAX) break;
    }
    aim = u * before;  // of a first pass, which picks nothing
    before = 0.0;
  }
  const int32_t token = pick_s != INT32_MAX ? pick_s : last_s;
  for (uint32_t j = tid; j <= a.K; j += kPickThreads)
    a.out[(uint64_t)b * (a.K + 1) + j] = j < m ? a.tokens[(uint64_t)b * a.K + j] : j == m ? token : -1;
}

hipError_t launch_verify_draft(const VerifyArgs& a, hipStream_t s) {
  if (!a.V || a.V > (1u << 30) || a.B > 65535) return hipErrorInvalidValue;
  if (!a.B) return hipSuccess;
  const dim3 grid((a.V + kVerifyChunk - 1) / kVerifyChunk, a.B);
#define OGKM_VERIFY(T)                                                               \
  do {                                                                               \
    hipLaunchKernelGGL((k_verify_sums<T>), grid, dim3(256), 0, s, a);                \
    hipLaunchKernelGGL((k_verify_pick<T>), dim3(a.B), dim3(kPickThreads), 0, s, a);  \
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
