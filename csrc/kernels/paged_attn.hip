// Attention of new tokens over a paged KV cache:
//   o_i = sum_{t <= pos_i} softmax_t(scale q_i . k_t) v_t,   pos_i = kv - n + i
// for row i of a request with n new rows and kv cached tokens (the new ones
// among them). One pass over the keys with a running maximum m and sum l; both
// products on the matrix cores.
//
// Layout of the two products. A request's rows of one kv head are its new
// tokens times the g query heads of the group (row r: token r / g, head r % g),
// so a key is read once for all of them. The scores are computed transposed,
// S^T = K Q^T (A: 16 or 32 keys, B: 16 or 32 rows), because then
//   - a lane owns ONE row: its maximum, sum and rescaling are per-lane values,
//     and a row's keys lie in its own registers and one or three other lanes';
//   - the accumulator's registers ARE the B operand of O^T = V^T P^T: an MFMA
//     contracts over keys in any order as long as A and B agree, so P goes
//     from the first product's accumulator into the second without a shuffle,
//     and V^T is read from LDS in the same key order by the transposing LDS
//     read (a 4 x 16 tile per 16 lanes).
// K and V rows go global -> registers -> LDS (the next tile's loads fly while
// this one is multiplied).
//
// Two bodies. `few` (up to 32 rows per kv head: single tokens, drafts) is bound
// by the KV bytes: each wave streams its own 32-key blocks through wave-private
// LDS without barriers, the waves join at the end. 64 tokens of 64 query and 8 kv
// heads at up to 2048 keys: 68 - 71 us; 4 tokens of 32 / 8 heads at up to 131071:
// 260 us, 5.6 TB/s of K and V. `many` (prompt chunks) is bound by the matrix cores:
// four waves of 32 rows share each tile of 64 keys (128 of 64 dims). One launch
// serves both kinds in a mixed batch. The key axis is split where rows are few;
// k_paged_combine joins the parts.
//
// Probabilities enter the second product in the element type; the row's sum takes
// them in f32. `few` multiplies with what that rounding left over as well (a second
// operand, 2 x 16 bits): its matrix cores wait for memory, and a single token gets
// what the contiguous cache's kernel gives, whose probabilities stay in f32. Error
// against f64 (norm of the difference over the norm) without / with it, and us: 64
// tokens of 64:8 heads at up to 2048 keys, bf16, 2.14e-3 / 1.66e-3 (1.66e-3 is the
// output's own rounding), 67.0 / 67.9; 4 x 1 at 131071, fp16, 2.84e-4 / 2.09e-4, 259
// / 260; 64 x 4 70B rows 77.7 / 81.3; 1 x 1 at 1025 keys 9.7 / 9.9; 4 x 1 at 1025,
// 64-wide, 9.0 / 9.7; single tokens beside chunks, up to 6 % of the call. `many` is
// bound by the matrix cores and keeps the type's bits: with the second operand 4096
// rows behind 4095 keys take 560 us for 415 (1.66e-3 for 2.35e-3), 12 x 511 + 36 x 1
// 64-wide 59 for 49 (2.07e-4 for 2.89e-4), 32 x 5 rows 35.7 for 31.3.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ogkm/elem.hpp"
#include "ogkm/kernels.hpp"
#include "ogkm/paged.hpp"

namespace ogkm {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
  typedef Vec<__bf16>::v8 v8;
  static constexpr uint32_t kInf = 0x7F80u;  // exponent bits
  static __device__ __forceinline__ f32x4_t m16(u32x4 a, u32x4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t m32(u32x4 a, u32x4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<_Float16> {
  typedef Vec<_Float16>::v8 v8;
  static constexpr uint32_t kInf = 0x7C00u;
  static __device__ __forceinline__ f32x4_t m16(u32x4 a, u32x4 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_t m32(u32x4 a, u32x4 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

// P is kept as 2^kShift p: an fp16 probability below 2^-14 would lose bits as a
// subnormal (bf16 has f32's range); with it that begins at 2^-22. The sum
// carries the same factor.
template <typename T>
constexpr float kShift = 0.f;
template <>
constexpr float kShift<_Float16> = 8.f;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typename Vec<T>::v2 v = {from_f32<T>(a), from_f32<T>(b)};
  return __builtin_bit_cast(uint32_t, v);
}
// What pack2 rounded away, as a second pair: the two add up to a and b but for the
// square of the type's half step (2^-16 of bf16, 2^-22 of fp16).
template <typename T>
__device__ __forceinline__ uint32_t pack2_rest(float a, float b, uint32_t packed) {
  const typename Vec<T>::v2 v = __builtin_bit_cast(typename Vec<T>::v2, packed);
  return pack2<T>(a - to_f32<T>(v[0]), b - to_f32<T>(v[1]));
}

// Any infinity or NaN among N x 8 elements? Two by an instruction: a small multiple of
// each, added up in f32, stays finite exactly if all are (64 of 2^128 2^-100, or 65504).
__device__ __forceinline__ float add_dot(Vec<__bf16>::v2 a, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(a, __builtin_bit_cast(Vec<__bf16>::v2, 0x0D800D80u), c, false);  // 2^-100
}
__device__ __forceinline__ float add_dot(Vec<_Float16>::v2 a, float c) {
  return __builtin_amdgcn_fdot2(a, __builtin_bit_cast(Vec<_Float16>::v2, 0x3C003C00u), c, false);  // 1
}
template <typename T, int N>
__device__ __forceinline__ bool any_nonfinite(const u32x4 (&x)[N]) {
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pair = x[i][j];  // a bit_cast of x[i][j] itself would read x[i][0]
      s[j] = add_dot(__builtin_bit_cast(typename Vec<T>::v2, pair), s[j]);
    }
  return !(fabsf((s[0] + s[1]) + (s[2] + s[3])) < __builtin_inff());
}

// V with infinities or NaNs in a tile that some row does not see whole (a probability
// of 0 times such a value would be NaN), and in every block of the few-row body (an
// infinity times what a probability's rounding left, 0 or of either sign). Such a value is taken out
// of V, and the first key that has one is kept for each dim and kind (NaN, +inf,
// -inf) in LDS: a row sees keys 0 .. pos, so it sees one exactly if pos is not
// before that key, and special() adds what it does to the row's sum.
constexpr int32_t kNever = INT32_MAX;
template <typename T, int HD>
__device__ __forceinline__ void take_special(u32x4* v8, int32_t key, uint32_t dim, int32_t* first_key) {
  u32x4 x = *v8;
  constexpr uint32_t inf = Mma<T>::kInf;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int s = 0; s < 32; s += 16) {
      const uint32_t v = (x[j] >> s) & 0xFFFFu;
      if ((v & inf) == inf) {
        const uint32_t kind = (v & 0x7FFFu) > inf ? 0u : v == inf ? 1u : 2u;
        atomicMin(first_key + kind * HD + dim + 2 * j + s / 16, key);  // LDS, integers: the order does not matter
        x[j] &= ~(0xFFFFu << s);
      }
    }
  *v8 = x;
}
template <int HD>
__device__ __forceinline__ float special(float o, int32_t pos, uint32_t dim, const int32_t* first_key) {
  if (pos >= first_key[dim]) o = __builtin_nanf("");
  if (pos >= first_key[HD + dim]) o += __builtin_inff();
  if (pos >= first_key[2 * HD + dim]) o -= __builtin_inff();
  return o;
}

// The 4 x 16 transposing LDS read: lane i of 16 gives the address of row i / 4,
// elements 4 (i % 4) .. + 3, and gets column i of the four rows.
__device__ __forceinline__ u32x2 read_tr(const uint16_t* p) {
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
  return __builtin_bit_cast(u32x2, v);
}

// LDS rows are padded instead of swizzled: every access is then one lane
// address plus a constant that fits the instruction, where XOR-ed chunks cost
// the compiler an address register each (122 spilled registers in the 32-row
// body). K: 16 bytes, the 8 lanes of a read phase take one chunk of 8 rows; V:
// 32 bytes, a transposing read takes 32 bytes of 4 rows. Both touch every bank
// once.
template <int HD>
constexpr int kKRow = HD + 8;
template <int HD>
constexpr int kVRow = HD + 16;
template <int HD>
constexpr int kKVRow = kKRow<HD> + kVRow<HD>;  // elements of LDS per key

// IEEE maximum: one v_maximum3_f32 takes three values (a NaN among them makes the
// result NaN, which a NaN score makes of its row anyway), where fmaxf quiets
// every operand first.
__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max_other_half(float x) {  // of lanes l and l ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t lo = r[0], hi = r[1];  // a bit_cast of r[1] itself would read r[0]
  return max2(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}

// What a sum over the maximum m counts for over the maximum mx >= m; a sum that
// saw only -inf (0 or NaN) keeps its value where nothing else is there.
__device__ __forceinline__ float scale_to(float m, float mx) {
  return m == mx ? 1.f : m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - mx);
}

// The wave's number, known to the compiler as uniform: bounds, page ids and
// addresses that follow from it stay in scalar registers.
__device__ __forceinline__ uint32_t wave_id() { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

struct Request {
  int32_t row0, n;       // first row in q, new rows
  int32_t kv, cap;       // cached tokens; kv > cap: the table row is too short
};
__device__ __forceinline__ Request request_of(const PagedAttnArgs& a, uint32_t b) {
  Request r;
  r.row0 = min(max(a.cu_q[b], 0), (int32_t)a.n);
  r.n = min(max(a.cu_q[b + 1], r.row0), (int32_t)a.n) - r.row0;
  r.kv = max(a.kv_lens[b], 0);
  r.cap = (int32_t)(a.width << a.page_shift);
  return r;
}

// Keys of a K / V tile of the many-row body: 16 KB of K and 16 KB of V. (64 keys of
// 64 dims: a barrier, a maximum and the addresses of half the work each.)
template <int HD>
constexpr int32_t kManyKeys = 8192 / HD;

// Keys of one split: whole tiles of the many-row body (they are whole blocks of
// the few-row body), so that no tile reaches into the next split's keys; at least
// kMinSplit, so that short requests use few of the launch's splits.
constexpr int32_t kMinSplit = 256;
template <int HD>
__device__ __forceinline__ int32_t split_keys(int32_t kv, uint32_t splits) {
  const int32_t per = (int32_t)(((uint32_t)kv + splits - 1) / splits);
  return max((per + kManyKeys<HD> - 1) & ~(kManyKeys<HD> - 1), kMinSplit);
}
__device__ __forceinline__ int32_t splits_used(int32_t kv, int32_t per) { return max((kv + per - 1) / per, 1); }

// ---------------------------------------------------------------- few rows

// What the waves of a workgroup leave for each other, behind their blocks in LDS.
template <int HD, int NB, int NW>
struct FewJoin {
  float wm[NW][16 * NB], wl[NW][16 * NB];
  int32_t first_key[NW][3 * HD];  // take_special; set only by a wave that met one
  uint32_t special[NW];
};
template <int HD, int NB, int NW>
constexpr uint32_t kFewLds = NW * 32 * kKVRow<HD> * 2 + sizeof(FewJoin<HD, NB, NW>);  // bytes

template <typename T, int HD, int NB, int NW>
__device__ __forceinline__ void few_body(const PagedAttnArgs& a, uint16_t* lds, uint32_t b, uint32_t kvh, uint32_t split) {
  constexpr int KS = HD / 32, DT = HD / 16, LD = HD / 32;  // k steps, dim tiles, loads per 16 rows
  constexpr int R = 16 * NB;
  const uint32_t lane = threadIdx.x & 63, wave = wave_id();
  const uint32_t col = lane & 15, quad = lane >> 4;
  const uint32_t g = a.hq / a.hkv;
  const Request rq = request_of(a, b);
  const int32_t rows = rq.n * (int32_t)g;
  if (rows == 0 || rows > (int32_t)a.plan.few_rows) return;
  const bool looped = rows > R;  // more rows than the host's bound: tile after tile, unsplit
  const int32_t kv = rq.kv > rq.cap ? 0 : rq.kv;
  const int32_t per = looped ? max(kv, 1) : split_keys<HD>(kv, a.plan.few_splits);
  const int32_t used = looped ? 1 : splits_used(kv, per);
  if ((int32_t)split >= used) return;
  const int32_t c0 = (int32_t)split * per, c1 = min(c0 + per, kv);
  // this wave's K block, then its V block; the lane's places in them
  uint16_t* kw = lds + wave * (32 * kKVRow<HD>) + (lane / (HD / 8)) * kKRow<HD> + (lane % (HD / 8)) * 8;
  uint16_t* vw = lds + wave * (32 * kKVRow<HD>) + 32 * kKRow<HD> + (lane / (HD / 8)) * kVRow<HD> + (lane % (HD / 8)) * 8;
  const uint16_t* kread = lds + wave * (32 * kKVRow<HD>) + col * kKRow<HD> + 8 * quad;
  const uint16_t* vread = lds + wave * (32 * kKVRow<HD>) + 32 * kKRow<HD> + (4 * quad + (col >> 2)) * kVRow<HD> + 4 * (col & 3);
  FewJoin<HD, NB, NW>& join = *reinterpret_cast<FewJoin<HD, NB, NW>*>(lds + NW * 32 * kKVRow<HD>);
  auto& wm = join.wm;
  auto& wl = join.wl;
  auto& first_key = join.first_key;
  auto& special_s = join.special;
  const uint16_t* kbase = a.pages + kvh * a.head_stride;
  const int32_t* table = a.table + b * a.table_ld;
  const float c = a.scale * 1.44269504088896340736f;  // scores in powers of two
  const int32_t blocks = (c1 - c0 + 31) >> 5;

  for (int32_t tile0 = 0; tile0 < rows; tile0 += R) {
    // this lane's rows, one per column block: the B operand and the last key each sees
    u32x4 qf[NB][KS];
    int32_t pos[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int32_t r = tile0 + nb * 16 + (int32_t)col;
      const bool in = r < rows;
      const uint32_t tok = in ? (uint32_t)r / g : 0u, h = in ? (uint32_t)r - tok * g : 0u;
      pos[nb] = in ? rq.kv - rq.n + (int32_t)tok : rq.kv - 1;
      const uint16_t* q = a.q + (uint64_t)(rq.row0 + tok) * a.q_stride + (kvh * g + h) * a.q_head_stride + 8 * quad;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        qf[nb][k] = *reinterpret_cast<const u32x4*>(q + 32 * k);
        if (!in) qf[nb][k] = u32x4{0u, 0u, 0u, 0u};
      }
    }
    // rows of this tile see keys up to here at least: blocks before it need no mask
    const int32_t first = rq.kv - rq.n + tile0 / (int32_t)g;
    f32x4_t o[NB][DT];
    float m[NB], l[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb] = -__builtin_inff();
      l[nb] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[nb][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    bool wave_special = false;
    // Page ids of this wave's next 32 blocks, one half block per lane (a page
    // holds at least 16 tokens), so that a block's addresses are wave-uniform.
    const int32_t mine = (blocks - (int32_t)wave + NW - 1) / NW;
    int32_t ids = 0;
    auto fetch_ids = [&](int32_t n0) {
      const int32_t t = c0 + ((n0 + (int32_t)(lane >> 1)) * NW + (int32_t)wave) * 32 + 16 * (int32_t)(lane & 1);
      ids = t < c1 ? table[t >> a.page_shift] : 0;
    };
    // The block ahead of the one multiplied, in registers.
    u32x4 kr[2 * LD], vr[2 * LD];
    bool missing[2] = {};
    auto load = [&](int32_t n) {
      if (n >= mine) return;
      if ((n & 31) == 0) fetch_ids(n);
      const int32_t t0 = c0 + (n * NW + (int32_t)wave) * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int32_t page = __builtin_amdgcn_readlane(ids, 2 * (n & 31) + h);
        const bool miss = (uint32_t)page >= a.num_pages;
        missing[h] = miss;
        if (miss) page = 0;
        const uint32_t row = (uint32_t)(t0 + 16 * h) & ((1u << a.page_shift) - 1u);
        const uint16_t* src = kbase + (uint64_t)page * a.page_stride + (uint64_t)row * HD;
#pragma unroll
        for (int j = 0; j < LD; ++j) kr[h * LD + j] = *reinterpret_cast<const u32x4*>(src + (j * 64 + lane) * 8);
#pragma unroll
        for (int j = 0; j < LD; ++j)
          vr[h * LD + j] = *reinterpret_cast<const u32x4*>(src + a.kv_stride + (j * 64 + lane) * 8);
      }
    };
    load(0);
    for (int32_t n = 0; n < mine; ++n) {
      const bool miss0 = missing[0], miss1 = missing[1];
      const int32_t t0 = c0 + (n * NW + (int32_t)wave) * 32;
      const bool masked = t0 + 31 > first;
      const bool odd = any_nonfinite<T>(vr);
#pragma unroll
      for (int j = 0; j < 2 * LD; ++j) {  // 512 / HD rows by each wave-wide store
        *reinterpret_cast<u32x4*>(kw + j * (512 / HD) * kKRow<HD>) = kr[j];
        *reinterpret_cast<u32x4*>(vw + j * (512 / HD) * kVRow<HD>) = vr[j];
      }
      if (__any(odd)) {
        if (!wave_special)
          for (uint32_t e = lane; e < 3 * HD; e += 64) first_key[wave][e] = kNever;
        wave_special = true;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int j = 0; j < 2 * LD; ++j)
          take_special<T, HD>(reinterpret_cast<u32x4*>(vw + j * (512 / HD) * kVRow<HD>),
                              t0 + j * (512 / HD) + (int32_t)(lane / (HD / 8)), lane % (HD / 8) * 8, first_key[wave]);
      }
      load(n + 1);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      // S^T: two tiles of 16 keys
      f32x4_t s[2][NB];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[t][nb] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const u32x4 ka = *reinterpret_cast<const u32x4*>(kread + t * 16 * kKRow<HD> + 32 * k);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) s[t][nb] = Mma<T>::m16(ka, qf[nb][k], s[t][nb]);
        }
      }
      u32x4 p[NB], rest[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float x[8];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = s[t][nb][r] * c;
            if (t ? miss1 : miss0) v = __builtin_nanf("");  // a page outside the pool
            x[4 * t + r] = v;
          }
        if (masked) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (t0 + 16 * t + 4 * (int32_t)quad + r > pos[nb]) x[4 * t + r] = -__builtin_inff();
        }
        float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m[nb], mx);
        if (__any(mn > m[nb])) {
          const float f = m[nb] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m[nb] - mn);
          // a row that saw only -inf so far has l = 0 or NaN: kept by l * 1
          const float fl = m[nb] == mn ? 1.f : f;
          l[nb] *= fl;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[nb][d] *= fl;
          m[nb] = mn;
        }
        const float base = (mn == -__builtin_inff() ? 0.f : mn) - kShift<T>;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = __builtin_amdgcn_exp2f(x[j] - base);
          l[nb] += x[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[nb][j] = pack2<T>(x[2 * j], x[2 * j + 1]);
          rest[nb][j] = pack2_rest<T>(x[2 * j], x[2 * j + 1], p[nb][j]);
        }
      }
      // O^T += V^T P^T, keys in the order of P's registers: 4 quad .. + 3 of each 16-key tile
      auto v_frag = [&](int d) {
        const u32x2 lo = read_tr(vread + 16 * d), hi = read_tr(vread + 16 * kVRow<HD> + 16 * d);
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
      };
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const u32x4 va = v_frag(d);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[nb][d] = Mma<T>::m16(va, p[nb], o[nb][d]);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) o[nb][d] = Mma<T>::m16(va, rest[nb], o[nb][d]);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    // Join the waves: maxima through LDS, then rounds in which the upper half of
    // the waves left is added to the lower, f32 in the K / V space.
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      l[nb] += __shfl_xor(l[nb], 16, 64);
      l[nb] += __shfl_xor(l[nb], 32, 64);
      if (quad == 0) {
        wm[wave][nb * 16 + col] = m[nb];
        wl[wave][nb * 16 + col] = l[nb];
      }
    }
    if (lane == 0) special_s[wave] = wave_special;
    __syncthreads();  // also: every wave is done with its blocks
    float big[NB], sum[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t r = nb * 16 + col;
      big[nb] = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < NW; ++w) big[nb] = fmaxf(big[nb], wm[w][r]);
      sum[nb] = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = wm[w][r] == -__builtin_inff() ? (big[nb] == wm[w][r] ? 1.f : 0.f)
                                                      : __builtin_amdgcn_exp2f(wm[w][r] - big[nb]);
        sum[nb] += f * wl[w][r];
        if ((uint32_t)w == wave)
#pragma unroll
          for (int d = 0; d < DT; ++d) o[nb][d] *= f;
      }
    }
    float* ox = reinterpret_cast<float*>(lds);  // [NW / 2][R][HD]; the lanes' own order, 16 bytes each
    auto put = [&](float* at) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4_t*>(at + ((nb * DT + d) * 64 + lane) * 4) = o[nb][d];
    };
    auto add = [&](const float* at) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int d = 0; d < DT; ++d) o[nb][d] += *reinterpret_cast<const f32x4_t*>(at + ((nb * DT + d) * 64 + lane) * 4);
    };
#pragma unroll 1
    for (uint32_t left = NW / 2; left; left /= 2) {
      if (wave >= left && wave < 2 * left) put(ox + (wave - left) * R * HD);
      __syncthreads();
      if (wave < left) add(ox + wave * R * HD);
      __syncthreads();
    }
    if (wave == 0) {
      for (int w = 0; w < NW; ++w)
        if (special_s[w])
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nb][d][e] = special<HD>(o[nb][d][e], pos[nb], 16 * d + 4 * quad + e, first_key[w]);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int32_t r = tile0 + nb * 16 + (int32_t)col;
        if (r >= rows) continue;
        const uint32_t tok = (uint32_t)r / g, h = (uint32_t)r - tok * g;
        if (used == 1) {
          float inv = 1.f / sum[nb];
          if (rq.kv > rq.cap) inv = __builtin_nanf("");
          uint16_t* dst = a.out + (uint64_t)(rq.row0 + tok) * a.out_stride + (uint64_t)(kvh * g + h) * HD + 4 * quad;
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            f32x4_t v = o[nb][d];
            // a row that sees nothing is 0; 0 / 0 of a row that saw only -inf is NaN
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = pos[nb] < 0 && rq.kv <= rq.cap ? 0.f : sum[nb] == 0.f ? __builtin_nanf("") : v[e] * inv;
            *reinterpret_cast<u32x2*>(dst + 16 * d) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
          }
        } else {
          const uint64_t at = (((uint64_t)b * a.hkv + kvh) * a.plan.few_splits + split) * R + nb * 16 + col;
          if (quad == 0) {
            a.part_ml[2 * at] = big[nb];
            a.part_ml[2 * at + 1] = sum[nb];
          }
#pragma unroll
          for (int d = 0; d < DT; ++d)
            *reinterpret_cast<f32x4_t*>(a.part_o + at * HD + 16 * d + 4 * quad) = o[nb][d];
        }
      }
    }
    if (looped) __syncthreads();  // wave 0 still reads what the next tile writes
  }
}

// ---------------------------------------------------------------- many rows
constexpr int kManyRows = 128;  // rows of a workgroup's tile: 4 waves of 32

// Tile x of all tiles of the requests with more than few_rows rows, a request's
// last tile first (of a prompt's tiles the last sees the most keys), the last
// request first. With more than one tile a CU the request with the most keys first
// instead, so that no long tile starts late or beside another. us in request order /
// so: 16 requests of 256 - 511 rows, 64-wide heads, at 512 - 2047 keys 66 / 57; 16 of
// 150 - 300 (8B heads) 123 / 109; 4 of 256 - 511 at 1024 - 4096 keys 125 / 105; 12 of
// 256 - 511 beside 36 single tokens 47 / 48 and 52 / 47, as the lengths fall. Every
// wave scans the request lengths by itself, 256 a round. Returns false past the end.
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& a, uint32_t x, uint32_t* b, int32_t* tile) {
  constexpr int E = 4;  // requests of a lane: top - 1 - E lane - e
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t g = a.hq / a.hkv;
  if (a.plan.many_sorted) {  // B <= 64: a lane has a request
    const bool is = lane < a.B;
    const int32_t end = a.cu_q[min(lane + 1, a.B)], begin = a.cu_q[min(lane, a.B)];
    const int32_t kv = is ? a.kv_lens[lane] : 0;
    const int32_t lo = min(max(begin, 0), (int32_t)a.n), hi = min(max(end, lo), (int32_t)a.n);
    const uint32_t rows = is ? (uint32_t)(hi - lo) * g : 0;
    const uint32_t tiles = rows > a.plan.few_rows ? (rows + kManyRows - 1) / kManyRows : 0;
    uint32_t before = 0;
    for (uint64_t left = __ballot(tiles > 0); left; left &= left - 1) {
      const int l = __builtin_ctzll(left);
      const int32_t other = __builtin_amdgcn_readlane(kv, l);
      const uint32_t its = (uint32_t)__builtin_amdgcn_readlane((int)tiles, l);
      before += other > kv || (other == kv && l < (int)lane) ? its : 0;
    }
    const uint64_t here = __ballot(before <= x && x - before < tiles);
    if (!here) return false;
    const int l = __builtin_ctzll(here);
    *b = (uint32_t)l;
    *tile = (int32_t)((uint32_t)__builtin_amdgcn_readlane((int)(before + tiles), l) - 1 - x);
    return true;
  }
  for (int32_t top = (int32_t)a.B; top > 0; top -= 64 * E) {
    const int32_t r0 = top - 1 - E * (int32_t)lane;
    int32_t cu[E + 1];  // of requests r0 + 1 - e; every index that exists is in bounds
#pragma unroll
    for (int e = 0; e <= E; ++e) cu[e] = a.cu_q[max(r0 + 1 - e, 0)];
    uint32_t upto[E], sum = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int32_t lo = min(max(cu[e + 1], 0), (int32_t)a.n), hi = min(max(cu[e], lo), (int32_t)a.n);
      const uint32_t rows = r0 - e >= 0 ? (uint32_t)(hi - lo) * g : 0;
      sum += rows > a.plan.few_rows ? (rows + kManyRows - 1) / kManyRows : 0;
      upto[e] = sum;
    }
    uint32_t before = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t y = __shfl_up(before, o, 64);
      if ((int)lane >= o) before += y;
    }
    const uint64_t past = __ballot(before > x);
    if (past) {
      const int l = __builtin_ctzll(past);
      const uint32_t from = (uint32_t)__builtin_amdgcn_readlane((int)(before - sum), l);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t end = from + (uint32_t)__builtin_amdgcn_readlane((int)upto[e], l);
        if (end > x) {
          *b = (uint32_t)(top - 1 - E * l - e);
          *tile = (int32_t)(end - 1 - x);
          return true;
        }
      }
    }
    x -= (uint32_t)__builtin_amdgcn_readlane((int)before, 63);
  }
  return false;
}

// Raise of a row's running maximum (in powers of two) that the accumulators do
// not follow: probabilities may reach 2^kLazy, and rescaling O becomes rare
// after the first tiles. fp16: 2^(kLazy + shift) stays below 65504.
constexpr float kLazy = 6.f;

// A wave owns 32 rows, the workgroup walks tiles of 8192 / HD keys in two LDS
// buffers: tile i + 1 flies into registers while tile i is multiplied, one barrier a tile
// (a buffer is written two tiles after it was read). 4096 rows behind 4095 cached
// keys of the 8B heads: 414 - 451 us on different cards, 995 - 914 TFLOP/s, where the
// library's 8192^3 product of such values reaches 1140 - 1230. The wave alternates between
// the matrix cores (1024 cycles a tile) and the vector ALU (1000, half of it
// exponentials); two workgroups a CU overlap them in part. Tried and not kept:
// 64 rows a wave (half the LDS reads, one wave per SIMD: 675 us); 32-key steps
// with the next scores beside the exponentials (444).

template <int HD>
constexpr uint32_t kManyLds = 2 * kManyKeys<HD> * kKVRow<HD> * 2 + (3 * HD + 1) * 4;  // bytes

template <typename T, int HD>
__device__ __forceinline__ void many_body(const PagedAttnArgs& a, uint16_t* lds, uint32_t x, uint32_t kvh, uint32_t split) {
  constexpr int KS = HD / 16, DT = HD / 32;        // k steps, 32-dim tiles
  constexpr int KT = kManyKeys<HD>, NT = KT / 32;  // keys and 32-key scores of a tile
  constexpr int LJ = KT * HD / 8 / 256;            // 16-byte loads of a thread per tile and tensor
  constexpr int kWindow = 1024 / KT;               // tiles whose groups of 16 keys fill a wave's lanes
  constexpr uint32_t kTile = KT * kKVRow<HD>;         // LDS elements of a K and V tile
  constexpr uint32_t kV = KT * kKRow<HD>;             // where its V begins
  const uint32_t lane = threadIdx.x & 63, wave = wave_id(), tid = threadIdx.x;
  const uint32_t col = lane & 31, half = lane >> 5;
  const uint32_t g = a.hq / a.hkv;
  uint32_t b;
  int32_t ti;
  if (!find_tile(a, x, &b, &ti)) return;
  const Request rq = request_of(a, b);
  const int32_t rows = rq.n * (int32_t)g, r0 = ti * kManyRows;
  const bool bad = rq.kv > rq.cap;
  // keys that any row of the tile sees, and this split's share
  const int32_t last = rq.kv - rq.n + (min(r0 + kManyRows, rows) - 1) / (int32_t)g;
  const int32_t kend = bad ? 0 : max(last + 1, 0);
  const int32_t per = split_keys<HD>(kend, a.plan.many_splits), used = splits_used(kend, per);
  if ((int32_t)split >= used) return;
  const int32_t c0 = (int32_t)split * per, c1 = min(c0 + per, kend);
  const uint16_t* kbase = a.pages + kvh * a.head_stride;
  const int32_t* table = a.table + b * a.table_ld;
  // scores in powers of two; the sign of the scale goes into q, so that the
  // largest product is the largest score
  const float c = fabsf(a.scale) * 1.44269504088896340736f;
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;

  const int32_t r = r0 + (int32_t)(wave * 32 + col);
  const bool in = r < rows;
  const uint32_t tok = in ? (uint32_t)r / g : 0u, h = in ? (uint32_t)r - tok * g : 0u;
  const int32_t pos = in ? rq.kv - rq.n + (int32_t)tok : last;
  u32x4 qf[KS];
  {
    const uint16_t* q = a.q + (uint64_t)(rq.row0 + tok) * a.q_stride + (kvh * g + h) * a.q_head_stride + 8 * half;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      qf[k] = *reinterpret_cast<const u32x4*>(q + 16 * k);
#pragma unroll
      for (int j = 0; j < 4; ++j) qf[k][j] = in ? qf[k][j] ^ flip : 0u;
    }
  }
  // of this wave's rows: the fewest and the most keys seen
  const int32_t w0 = r0 + (int32_t)wave * 32, w1 = min(w0 + 32, rows) - 1;
  const int32_t wfirst = rq.kv - rq.n + w0 / (int32_t)g;
  const int32_t wlast = w0 < rows ? rq.kv - rq.n + w1 / (int32_t)g : -1;

  f32x16_t o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m = -__builtin_inff(), l = 0.f;  // m: what the accumulators are scaled by, in units of c

  // the lane's places in a tile
  const uint32_t kw = tid / (HD / 8) * kKRow<HD> + tid % (HD / 8) * 8, vw = kV + tid / (HD / 8) * kVRow<HD> + tid % (HD / 8) * 8;
  const uint32_t kread = col * kKRow<HD> + 8 * half;
  const uint32_t vread = kV + (4 * half + ((lane & 15) >> 2)) * kVRow<HD> + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  const uint32_t mine = (tid / (HD / 8)) % 16 * HD + tid % (HD / 8) * 8;  // in its group of 16 keys

  // Where the lane's group of 16 keys (one page) begins, for kWindow tiles. A group
  // whose page is outside the pool reads page 0; the first such key makes the
  // rows that see it NaN.
  int32_t first_missing = rq.kv > rq.cap ? 0 : kNever;
  uint32_t at_lo = 0, at_hi = 0;
  auto find_groups = [&](int32_t i) {
    const int32_t t = c0 + i * KT + 16 * (int32_t)lane;
    int32_t page = t < c1 ? table[t >> a.page_shift] : 0;
    const uint64_t outside = __ballot((uint32_t)page >= a.num_pages);
    if (outside) first_missing = min(first_missing, c0 + i * KT + 16 * (int32_t)__builtin_ctzll(outside));
    if ((uint32_t)page >= a.num_pages) page = 0;
    const uint64_t at = (uint64_t)page * a.page_stride + (uint64_t)((uint32_t)t & ((1u << a.page_shift) - 1u)) * HD;
    at_lo = (uint32_t)at;
    at_hi = (uint32_t)(at >> 32);
  };
  u32x4 kr[LJ], vr[LJ];
  auto load = [&](int32_t i) {
    if (i % kWindow == 0) find_groups(i);
#pragma unroll
    for (int j = 0; j < LJ; ++j) {
      const uint32_t grp = KT / 16 * (i % kWindow) + (j * 256 + wave * 64) / (HD / 8) / 16;  // wave-uniform
      const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)at_lo, grp) |
                          (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)at_hi, grp) << 32;
      kr[j] = *reinterpret_cast<const u32x4*>(kbase + at + mine);
      vr[j] = *reinterpret_cast<const u32x4*>(kbase + a.kv_stride + at + mine);
    }
  };
  const int32_t tiles = (c1 - c0 + KT - 1) / KT;
  const int32_t first = rq.kv - rq.n + r0 / (int32_t)g;  // of the whole tile of rows
  int32_t* first_key = reinterpret_cast<int32_t*>(lds + 2 * kTile);  // [3 * HD], take_special
  int32_t& special_s = first_key[3 * HD];
  for (uint32_t e = tid; e < 3 * HD; e += 256) first_key[e] = kNever;
  if (tid == 0) special_s = 0;
  if (tiles > 0) load(0);
  __syncthreads();
  for (int32_t i = 0; i < tiles; ++i) {
    const int32_t t0 = c0 + i * KT;
    uint16_t* buf = lds + (i & 1) * kTile;
    const bool tile_masked = t0 + KT - 1 > first;
    const bool odd = tile_masked && any_nonfinite<T>(vr);
#pragma unroll
    for (int j = 0; j < LJ; ++j) {
      *reinterpret_cast<u32x4*>(buf + kw + j * (2048 / HD) * kKRow<HD>) = kr[j];
      *reinterpret_cast<u32x4*>(buf + vw + j * (2048 / HD) * kVRow<HD>) = vr[j];
    }
    if (odd) {
      special_s = 1;
#pragma unroll 1
      for (int j = 0; j < LJ; ++j)
        take_special<T, HD>(reinterpret_cast<u32x4*>(buf + vw + j * (2048 / HD) * kVRow<HD>),
                            t0 + j * (2048 / HD) + (int32_t)(tid / (HD / 8)), tid % (HD / 8) * 8, first_key);
    }
    if (i + 1 < tiles) load(i + 1);
    // the other buffer's readers passed the barrier of the tile before
    __syncthreads();
    if (t0 > wlast) continue;  // none of this wave's rows sees the tile

    // Between the barrier and the last product a wave goes before those that load
    // and store (430 -> 421 us for the 4096 rows, 52 -> 49 for 12 x 400 64-wide).
    __builtin_amdgcn_s_setprio(1);
    f32x16_t s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k)
        s[t] = Mma<T>::m32(*reinterpret_cast<const u32x4*>(buf + kread + t * 32 * kKRow<HD> + 16 * k), qf[k], s[t]);
    }
    // six operands ahead of the products: an LDS read takes longer than one
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int k = 0; k < NT * KS - 6; ++k) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 6, 0);
    // register e of s[t] is key 32 t + 8 (e / 4) + 4 half + e % 4
    if (t0 + KT - 1 > wfirst) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (t0 + 32 * t + 8 * (e / 4) + 4 * (int32_t)half + e % 4 > pos) s[t][e] = -__builtin_inff();
    }
    float mx = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < NT; t += 2)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = max2(max2(mx, s[t][e]), s[t + 1][e]);
    mx = max_other_half(mx) * c;
    if (__any(mx > m + kLazy) || i == 0) {
      const float mn = max2(m, mx);
      const float f = m == mn ? 1.f : m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
      m = mn;
    }
    const float base = (m == -__builtin_inff() ? 0.f : m) - kShift<T>;
    // Probabilities of keys 16 kt .. (registers 8 (kt % 2) .. of s[kt / 2]) as a B operand
    auto exponentials = [&](int kt) {
      u32x4 p;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[kt / 2][8 * (kt % 2) + 2 * e], c, -base));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[kt / 2][8 * (kt % 2) + 2 * e + 1], c, -base));
        l += p0 + p1;
        p[e] = pack2<T>(p0, p1);
      }
      return p;
    };
    // V^T operand of dims 32 d .., keys 16 kt ..: two 16-dim halves by lane group
    auto v_frag = [&](int d, int kt) {
      const uint16_t* at = buf + vread + 16 * kt * kVRow<HD> + 32 * d;
      const u32x2 lo = read_tr(at), hi = read_tr(at + 8 * kVRow<HD>);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    // The products of one group of 16 keys run beside the exponentials and the
    // operand reads of the next.
    u32x4 va[2][DT], p[2];
#pragma unroll
    for (int d = 0; d < DT; ++d) va[0][d] = v_frag(d, 0);
    p[0] = exponentials(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kt = 0; kt < 2 * NT; ++kt) {
      if (kt + 1 < 2 * NT) {
#pragma unroll
        for (int d = 0; d < DT; ++d) va[(kt + 1) & 1][d] = v_frag(d, kt + 1);
        p[(kt + 1) & 1] = exponentials(kt + 1);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] = Mma<T>::m32(va[kt & 1][d], p[kt & 1], o[d]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        __builtin_amdgcn_sched_group_barrier(0x002, 10 / DT, 1);
        __builtin_amdgcn_sched_group_barrier(0x400, 8 / DT, 1);
        __builtin_amdgcn_sched_group_barrier(0x002, 10 / DT, 1);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  }
  l += __shfl_xor(l, 32, 64);
  if (!in) return;
  if (pos >= first_missing) l = __builtin_nanf("");
  if (tiles > 0 && special_s)  // set before the last tile's barrier
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        o[d][e] = special<HD>(o[d][e], pos, 32 * d + 8 * (e / 4) + 4 * half + e % 4, first_key);
  if (used == 1) {
    // a row that sees nothing is 0; one that saw only -inf is NaN
    const float inv = pos < 0 && !bad ? 0.f : l == 0.f ? __builtin_nanf("") : 1.f / l;
    uint16_t* dst = a.out + (uint64_t)(rq.row0 + tok) * a.out_stride + (uint64_t)(kvh * g + h) * HD + 4 * half;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        *reinterpret_cast<u32x2*>(dst + 32 * d + 2 * e) = u32x2{pack2<T>(o[d][e] * inv, o[d][e + 1] * inv),
                                                                pack2<T>(o[d][e + 2] * inv, o[d][e + 3] * inv)};
      }
  } else {
    const uint64_t at = a.plan.few_part + (((uint64_t)x * a.hkv + kvh) * a.plan.many_splits + split) * kManyRows + wave * 32 + col;
    if (half == 0) {
      a.part_ml[2 * at] = m;
      a.part_ml[2 * at + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4_t*>(a.part_o + at * HD + 32 * d + 2 * e + 4 * half) =
            f32x4_t{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
  }
}

// Two column blocks of 128 dims take 346 registers where a CU holds one workgroup;
// with two (256 registers) fewer LDS reads were in flight and 40 registers spilled.
// us with two / with one: 16 requests of 4 tokens, 64 query and 8 kv heads, at up to
// 2048 keys 34.6 / 30.0, 64 of them 94 / 81, 1 at 65535 57.5 / 53.7. (The other shapes
// are not faster with one, and two blocks ahead in registers, 424 of them, lost
// another 2 - 6.)
template <int HD, int NB>
constexpr bool kWideFew = HD == 128 && NB == 2;

template <typename T, int HD, int NB, int NW>
__global__ void __launch_bounds__(64 * NW, (kWideFew<HD, NB> ? 1 : 2)) k_paged_few(PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[kFewLds<HD, NB, NW> / 2];
  few_body<T, HD, NB, NW>(a, lds, blockIdx.z, blockIdx.x, blockIdx.y);
}

// Both kinds of requests in one launch: the long tiles first, then the few-row
// requests, which fill in beside them.
template <typename T, int HD, int NB>
__global__ void __launch_bounds__(256, 2) k_paged_mixed(PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[std::max(kFewLds<HD, NB, 4>, kManyLds<HD>) / 2];  // 2 fit a CU
  uint32_t i = blockIdx.x;
  const uint32_t kvh = i % a.hkv;  // a head's workgroups share their K and V, and with 8 heads an XCD's L2
  i /= a.hkv;
  const uint32_t many = a.plan.many_tiles * a.plan.many_splits;
  if (i < many) {
    many_body<T, HD>(a, lds, i / a.plan.many_splits, kvh, i % a.plan.many_splits);
  } else {
    i -= many;
    few_body<T, HD, NB, 4>(a, lds, i / a.plan.few_splits, kvh, i % a.plan.few_splits);
  }
}

// Joins the splits. A unit is a tile of many rows, or the rows of a request of
// few; the units' first workgroups are those of the tiles. A thread takes four
// dims of a row and a slice of the splits (at most kSlices), four splits' loads in
// flight, with a running maximum; the slices meet in LDS.
constexpr uint32_t kSlices = 16;
__host__ __device__ constexpr uint32_t join_slices(uint32_t splits) {
  uint32_t z = 1;
  while (z < kSlices && 4 * z < splits) z *= 2;
  return z;
}
// Workgroups of a unit of `rows` rows (the host's bound; what lies beyond it is
// taken in further rounds): one round, but no more than 2048 workgroups in all.
uint32_t join_parts(uint64_t rows, uint32_t hd, uint32_t splits, uint64_t units) {
  const uint64_t all = (rows * (hd / 4) * join_slices(splits) + 255) / 256;
  return (uint32_t)std::max<uint64_t>(std::min<uint64_t>(all, 2048 / std::max<uint64_t>(units, 1)), 1);
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) k_paged_combine(PagedAttnArgs a, uint32_t many_parts, uint32_t few_parts) {
  __shared__ f32x4_t slice_o[256];
  __shared__ float slice_m[256], slice_l[256];
  const uint32_t kvh = blockIdx.y;
  const uint32_t g = a.hq / a.hkv;
  const uint32_t many_blocks = a.plan.many_splits > 1 ? a.plan.many_tiles * many_parts : 0;
  uint32_t b, splits, R, part, parts;
  int32_t r0, keys;  // first row of the unit in its request, keys that were split
  uint64_t at;
  Request rq;
  if (blockIdx.x < many_blocks) {
    parts = many_parts;
    const uint32_t x = blockIdx.x / parts;
    part = blockIdx.x % parts;
    int32_t ti;
    if (!find_tile(a, x, &b, &ti)) return;
    rq = request_of(a, b);
    r0 = ti * kManyRows;
    keys = max(rq.kv - rq.n + (min(r0 + kManyRows, rq.n * (int32_t)g) - 1) / (int32_t)g + 1, 0);
    splits = a.plan.many_splits;
    R = kManyRows;
    at = a.plan.few_part + ((uint64_t)x * a.hkv + kvh) * splits * R;
  } else {
    const uint32_t i = blockIdx.x - many_blocks;
    R = 16 * a.plan.few_blocks;
    splits = a.plan.few_splits;
    parts = few_parts;
    b = i / parts;
    part = i % parts;
    rq = request_of(a, b);
    if (rq.n * (int32_t)g > (int32_t)R) return;
    r0 = 0;
    keys = rq.kv;
    at = ((uint64_t)b * a.hkv + kvh) * splits * R;
  }
  if (rq.kv > rq.cap) return;
  const int32_t used = splits_used(keys, split_keys<HD>(keys, splits));
  if (used == 1) return;
  const uint32_t items = min((uint32_t)(rq.n * (int32_t)g - r0), R) * (HD / 4);
  const uint32_t slices = join_slices(splits), per = 256 / slices;
  const uint32_t slice = threadIdx.x / per, own = threadIdx.x % per;
  for (uint32_t first = part * per; first < items; first += parts * per) {
    const uint32_t item = first + own, rr = item / (HD / 4), d = item % (HD / 4) * 4;
    const bool in = item < items;
    float big = -__builtin_inff(), sum = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    if (in) {
      for (uint32_t s = slice; s < (uint32_t)used; s += 4 * slices) {
        float m[4], l[4];
        f32x4_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t i = at + rr + (uint64_t)min(s + e * slices, (uint32_t)used - 1) * R;
          m[e] = a.part_ml[2 * i];
          l[e] = a.part_ml[2 * i + 1];
          x[e] = *reinterpret_cast<const f32x4_t*>(a.part_o + i * HD + d);
        }
        float mx = big;
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = max2(mx, m[e]);
        const float old = scale_to(big, mx);
        sum *= old;
        o *= old;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (s + e * slices < (uint32_t)used) {
            const float f = scale_to(m[e], mx);
            sum += f * l[e];
            o += f * x[e];
          }
        big = mx;
      }
    }
    if (slices > 1) {
      __syncthreads();  // the slices of the round before are read
      slice_o[threadIdx.x] = o;
      slice_m[threadIdx.x] = big;
      slice_l[threadIdx.x] = sum;
      __syncthreads();
      if (slice == 0) {
        float mx = big;
        for (uint32_t z = 1; z < slices; ++z) mx = max2(mx, slice_m[z * per + own]);
        const float f0 = scale_to(big, mx);
        sum *= f0;
        o *= f0;
        for (uint32_t z = 1; z < min(slices, (uint32_t)used); ++z) {
          const float f = scale_to(slice_m[z * per + own], mx);
          sum += f * slice_l[z * per + own];
          o += f * slice_o[z * per + own];
        }
      }
    }
    if (!in || slice) continue;
    const uint32_t r = (uint32_t)r0 + rr, tok = r / g, h = r - tok * g;
    const float inv = rq.kv - rq.n + (int32_t)tok < 0 ? 0.f : 1.f / sum;
    uint16_t* out = a.out + (uint64_t)(rq.row0 + tok) * a.out_stride + (uint64_t)(kvh * g + h) * HD + d;
    // sum 0: the row saw only scores of -inf, 0 / 0
    if (sum == 0.f && inv != 0.f) o = f32x4_t{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
    *reinterpret_cast<u32x2*>(out) = u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
  }
}

template <typename T, int HD, int NB>
hipError_t launch_attn(const PagedAttnArgs& a, hipStream_t s) {
  const PagedAttnPlan& p = a.plan;
  if (p.many_tiles) {
    const uint64_t wgs = ((uint64_t)p.many_tiles * p.many_splits + (uint64_t)a.B * p.few_splits) * a.hkv;
    if (wgs >= (1u << 24)) return hipErrorInvalidValue;  // threads of a grid stay below 2^32
    hipLaunchKernelGGL((k_paged_mixed<T, HD, NB>), dim3((uint32_t)wgs), dim3(256), 0, s, a);
  } else {
    const dim3 grid(a.hkv, p.few_splits, a.B);
    if constexpr (!kWideFew<HD, NB>)
      if (p.few_waves == 8) {
        hipLaunchKernelGGL((k_paged_few<T, HD, NB, 8>), grid, dim3(512), 0, s, a);
        return hipGetLastError();  // never split
      }
    hipLaunchKernelGGL((k_paged_few<T, HD, NB, 4>), grid, dim3(256), 0, s, a);
  }
  const uint64_t many_units = p.many_splits > 1 ? p.many_tiles : 0, few_units = p.few_splits > 1 ? a.B : 0;
  const uint64_t units = (many_units + few_units) * a.hkv;
  const uint32_t many_parts = join_parts(std::min<uint32_t>(p.most_rows, kManyRows), HD, p.many_splits, units);
  const uint32_t few_parts = join_parts(std::min<uint32_t>(p.most_rows, 16 * NB), HD, p.few_splits, units);
  const uint64_t groups = many_units * many_parts + few_units * few_parts;
  if (groups >= (1u << 24)) return hipErrorInvalidValue;
  if (groups)
    hipLaunchKernelGGL((k_paged_combine<T, HD>), dim3((uint32_t)groups, a.hkv), dim3(256), 0, s, a, many_parts, few_parts);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_attn_of(const PagedAttnArgs& a, hipStream_t s) {
  if (a.hd == 128) return a.plan.few_blocks == 1 ? launch_attn<T, 128, 1>(a, s) : launch_attn<T, 128, 2>(a, s);
  return a.plan.few_blocks == 1 ? launch_attn<T, 64, 1>(a, s) : launch_attn<T, 64, 2>(a, s);
}

}  // namespace

PagedAttnPlan paged_attn_plan(uint32_t n, uint32_t B, uint32_t hq, uint32_t hkv, uint32_t hd, uint32_t max_q,
                              uint32_t max_kv) {
  PagedAttnPlan p{};
  const uint64_t g = hq / hkv, most = std::min(max_q, n) * g;  // rows of a request, at most
  const uint64_t heads = hkv, key_splits = std::max<uint64_t>((max_kv + kMinSplit - 1) / kMinSplit, 1);
  // Up to 32 rows: the few-row body. (With 4 column blocks, up to 64, it needs all
  // 512 registers: 32 x 5 drafted rows of 8 heads at up to 8191 keys took 48 us,
  // the other body's half-empty tiles take 38.)
  const bool only_few = most <= 32;
  p.most_rows = (uint32_t)most;
  const uint64_t few = only_few ? most : g;  // rows that the few-row body is laid out for
  p.few_blocks = few <= 16 ? 1 : 2;
  p.many_splits = 1;
  if (only_few) {
    p.few_rows = INT32_MAX;  // a request beyond the host's bound is taken tile by tile
  } else {
    // 0 rows where one token already takes more
    p.few_rows = g <= 32 ? 16 * p.few_blocks : 0;
    // m requests of r_i rows have at most floor((sum r_i + 127 m) / 128) tiles
    const uint64_t at_most = std::min<uint64_t>(B, n * g / (p.few_rows + 1));
    p.many_tiles = (uint32_t)((n * g + (kManyRows - 1) * at_most) / kManyRows);
    // The number of splits with the least expected time, in us: a workgroup's share of
    // the keys (a prompt's rows see about three quarters of its own) at what a tile of
    // them takes alone on its CU, longer by half beside a second workgroup; the join;
    // partial results written and read at 7 TB/s (they stay in the caches). us measured
    // with 1 / 2 / 3 / 4 / 6 / 8 / 12 splits, the chosen one in brackets:
    //   512 rows of a prompt's start, 8B heads      [18] 24 26 26 28 32 36
    //   2 x 42 rows behind 1508, 24:8 heads          38 27 22 20 18 [18] 18
    //   25 x 58 - 116 rows of 8:1 at up to 545      [23] 28 26 36 31 53 46
    //   2 x 220 rows behind 2198, 16:4, 64 wide      36 25 22 20 [20] 21 22
    //   1024 rows behind 7168, 8B heads             182 [148] 157 156
    // and 32 x 5 rows of 8:1 at up to 8191 37 / 33 / 31 with 6 / 8 / 12.
    const uint64_t wgs = std::max<uint64_t>(p.many_tiles * heads, 1);
    const double keys = std::max<double>(max_kv - std::min(max_q, n) / 4.0, 1.0);
    double best = 0.0;
    for (uint32_t splits = 1; splits <= std::min<uint64_t>(key_splits, 64); ++splits) {
      const double load = (double)wgs * splits / 256.0;  // workgroups a CU
      double us = keys * (hd == 64 ? 0.010 : 0.0165) / splits * (load <= 1 ? 1.0 : load <= 2 ? 0.5 + 0.5 * load : 0.75 * load);
      if (splits > 1) us += 3.0 + (double)n * hq * splits * (hd + 2) * 8 / 7e6;
      if (splits == 1 || us < best) {
        best = us;
        p.many_splits = splits;
      }
    }
    // (32 short requests in 13 splits: 31 us in request order, 33 sorted)
    p.many_sorted = B > 1 && B <= 64 && p.many_splits <= 2 && wgs * p.many_splits > 256;
  }
  // A workgroup a CU: four waves with a block each in flight draw what HBM gives.
  // us at 128 / 256 / 512 / 1024 workgroups, ragged lengths: 4 requests of up to 131071
  // keys 332 / 235 / 198 / 196, 16 of 4096 41.5 / 34.6 / 34.6 / 33.4, 64 of 2048 (70B
  // heads) 69.7 / 69.5 / 69.5 / 75.1, 4 of 8192 27.6 / 21.5 / 19.9 / 22.9; 16 x 4 rows
  // of 70B heads at 2048 39 / 30 / 36 / 47, 1 x 4 at 65535 70 / 54 / 60 / 76. Half of
  // that beside longer requests, whose tiles fill the CUs too; us at 128 / 256: 13
  // single tokens beside 4 chunks of 155 rows at up to 1585 keys, 64-wide, 22.3 / 20.9,
  // 36 beside 12 of 511 at 2047 50.1 / 48.6, 7 beside 14 of 351 at 1046 20.2 / 23.1,
  // 35 beside 4 of 394 at 1234, 24:8 heads, 45.3 / 45.2 (a token each of 4 requests at
  // 131071 and a chunk: 113, and 142 at 64 workgroups).
  // Not at all for one request, which the bound says has more rows (4096 rows of a
  // prompt behind 4095 keys: 5 us of joining nothing).
  const uint64_t wgs = std::max<uint64_t>(B * heads, 1), few_wgs = only_few ? 256 : B > 1 ? 128 : 1;
  p.few_splits = (uint32_t)std::min<uint64_t>((few_wgs + wgs - 1) / wgs, key_splits);
  // Short contexts of few requests: eight waves and no second launch. us a call with it
  // / with splits (on the GPU alone): one request of the 8B heads at 512 keys 9.8 / 13.5
  // (9.4 / 9.4), at 1025 13.6 / 13.5 (13.2 / 9.9), at 1536 16.9 / 13.6 (16.5 / 9.9); 4
  // requests of 64-wide heads at 1025 10.0 / 13.7 (9.7 / 8.8). (Two column blocks of 128
  // dims would spill: 21 us at 700 keys.)
  p.few_waves = 4;
  if (only_few && p.few_splits > 1 && (uint64_t)max_kv * hd <= 96 * 1024 && (p.few_blocks == 1 || hd == 64)) {
    p.few_waves = 8;
    p.few_splits = 1;
  }
  p.few_part = p.few_splits > 1 ? wgs * p.few_splits * 16 * p.few_blocks : 0;
  p.part_rows = p.few_part + (p.many_splits > 1 ? p.many_tiles * heads * p.many_splits * kManyRows : 0);
  return p;
}

hipError_t launch_paged_attn(const PagedAttnArgs& a, hipStream_t s) {
  if (!a.hkv || a.hq % a.hkv || (a.hd != 64 && a.hd != 128) || a.page_shift < 4 || a.page_shift > 8 || !a.plan.few_splits ||
      a.hkv > 65535 || a.plan.few_splits > 65535 || a.B > 65535)
    return hipErrorInvalidValue;
  if (!a.n || !a.B) return hipSuccess;
  return a.elem == ELEM_F16 ? launch_attn_of<_Float16>(a, s) : launch_attn_of<__bf16>(a, s);
}

}  // namespace ogkm
