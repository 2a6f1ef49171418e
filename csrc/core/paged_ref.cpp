// CPU references of the paged-serving ops (csrc/kernels/paged_ops.hip,
// paged_attn.hip, speculative.hip) for the fake backend and tests: the same
// layouts, bounds and outcomes, in f64 where a border decides.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "ogkm/paged.hpp"

namespace ogkm {

static inline float bf2f(uint16_t b) {
  uint32_t u = (uint32_t)b << 16;
  float f;
  memcpy(&f, &u, 4);
  return f;
}
static inline uint16_t f2bf(float f) {
  uint32_t u;
  memcpy(&u, &f, 4);
  if ((u & 0x7F800000u) == 0x7F800000u && (u & 0x7FFFFFu)) return (uint16_t)((u >> 16) | 0x40u);
  u += 0x7FFFu + ((u >> 16) & 1u);
  return (uint16_t)(u >> 16);
}
// fp16 by hand: not every host compiler that builds this file has the type.
static inline float h2f(uint16_t b) {
  const uint32_t sign = (uint32_t)(b & 0x8000u) << 16, rest = b & 0x7FFFu;
  if (rest < 0x400u) {  // zero, subnormal
    const float f = (float)rest * 0x1p-24f;
    return sign ? -f : f;
  }
  const uint32_t u = sign | (rest >= 0x7C00u ? 0x7F800000u | (rest & 0x3FFu) << 13 : (rest << 13) + (112u << 23));
  float f;
  memcpy(&f, &u, 4);
  return f;
}
static inline uint16_t f2h(float f) {  // to nearest, ties to even
  uint32_t u;
  memcpy(&u, &f, 4);
  const uint16_t sign = (uint16_t)((u >> 16) & 0x8000u);
  u &= 0x7FFFFFFFu;
  if (u > 0x7F800000u) return (uint16_t)(sign | 0x7E00u | ((u >> 13) & 0x3FFu));
  if (u >= 0x477FF000u) return (uint16_t)(sign | 0x7C00u);  // 65520 and above
  if (u < 0x38800000u) return (uint16_t)(sign | (uint32_t)std::nearbyint(std::fabs(f) * 0x1p24f));  // below 2^-14
  u += 0xFFFu + ((u >> 13) & 1u);
  return (uint16_t)(sign | ((u - (112u << 23)) >> 13));
}
static inline float load16(uint16_t b, uint32_t elem) { return elem == ELEM_F16 ? h2f(b) : bf2f(b); }
static inline uint16_t store16(float f, uint32_t elem) { return elem == ELEM_F16 ? f2h(f) : f2bf(f); }

void paged_plan_cpu(const PlanArgs& a) {
  const int64_t P = 1ll << a.page_shift;
  const int64_t start = std::min<int64_t>(std::max(a.free_start[0], 0), a.n_free);
  int64_t end = 0, upto = 0, taken = 0;
  a.cu_q[0] = 0;
  std::fill(a.positions, a.positions + a.n_tokens, -1);
  std::fill(a.slots, a.slots + a.n_tokens, -1);
  for (uint32_t b = 0; b < a.B; ++b) {
    const int64_t fresh = std::max(a.new_lens[b], 0), kv = std::max(a.kv_lens[b], 0);
    const int64_t have = std::min<int64_t>(std::max(a.page_counts[b], 0), a.width);
    const int64_t row0 = std::min<int64_t>(end, a.n_tokens);
    end += fresh;
    const int64_t total = (kv + fresh + P - 1) >> a.page_shift;
    const bool fits = total <= (int64_t)a.width && end <= (int64_t)a.n_tokens;
    const int64_t need = fits ? std::max<int64_t>(total - have, 0) : 0;
    const int64_t first = start + upto;
    upto += need;
    const bool granted = fits && (need == 0 || start + upto <= (int64_t)a.n_free);
    a.cu_q[b + 1] = (int32_t)std::min<int64_t>(end, a.n_tokens);
    a.granted[b] = granted;
    a.kv_out[b] = (int32_t)(granted ? kv + fresh : kv);
    a.counts_out[b] = (int32_t)(granted ? std::max(have, total) : have);
    if (!granted) continue;
    taken += need;
    int32_t* row = a.table + (uint64_t)b * a.table_ld;
    for (int64_t j = 0; j < need; ++j) row[have + j] = a.free_pages[first + j];
    for (int64_t t = 0; t < fresh; ++t) {
      const int64_t pos = kv + t, page = row[pos >> a.page_shift];
      a.positions[row0 + t] = (int32_t)pos;
      a.slots[row0 + t] = page < 0 || page > (INT32_MAX >> a.page_shift) ? -1 : (int32_t)((page << a.page_shift) + (pos & (P - 1)));
    }
  }
  a.free_out[0] = (int32_t)(start + taken);
}

void paged_rope_cpu(const PagedRopeArgs& a) {
  const uint32_t half = a.hd / 2, heads = a.hq + 2 * a.hkv;
  const uint32_t mask = (1u << a.page_shift) - 1;
  for (uint32_t t = 0; t < a.n; ++t) {
    const int32_t pos = a.positions[t], slot = a.slots[t];
    const bool inside = slot >= 0 && ((uint32_t)slot >> a.page_shift) < a.num_pages;
    for (uint32_t h = 0; h < heads; ++h)
      for (uint32_t i = 0; i < half; ++i) {
        const uint16_t* src = a.qkv + t * a.ldqkv + (uint64_t)h * a.hd;
        uint16_t o1 = src[i], o2 = src[i + half];
        if (h < a.hq + a.hkv) {
          float c = NAN, s = NAN;
          if (pos >= 0 && (uint32_t)pos < a.max_pos) {
            c = a.cos[(uint64_t)pos * half + i];
            s = a.sin[(uint64_t)pos * half + i];
          }
          const float x1 = load16(o1, a.elem), x2 = load16(o2, a.elem);
          o1 = store16(pos < 0 ? 0.f : x1 * c - x2 * s, a.elem);
          o2 = store16(pos < 0 ? 0.f : x2 * c + x1 * s, a.elem);
        }
        uint16_t* dst;
        if (h < a.hq) {
          dst = a.q_out + ((uint64_t)t * a.hq + h) * a.hd;
        } else {
          if (!inside || pos < 0) continue;
          const uint32_t kv = h < a.hq + a.hkv ? 0 : 1;
          dst = a.pages + kv * a.kv_stride + ((uint32_t)slot >> a.page_shift) * a.page_stride +
                (h - a.hq - kv * a.hkv) * a.head_stride + (uint64_t)((uint32_t)slot & mask) * a.hd;
        }
        dst[i] = o1;
        dst[i + half] = o2;
      }
  }
}

void paged_attn_cpu(const PagedAttnArgs& a) {
  const uint32_t g = a.hq / a.hkv, P = 1u << a.page_shift;
  const int64_t cap = (int64_t)a.width << a.page_shift;
  std::vector<double> sc, o(a.hd);
  for (uint32_t b = 0; b < a.B; ++b) {
    const int64_t lo = std::min<int64_t>(std::max(a.cu_q[b], 0), a.n);
    const int64_t hi = std::min<int64_t>(std::max<int64_t>(a.cu_q[b + 1], lo), a.n);
    const int64_t kv = std::max(a.kv_lens[b], 0);
    const int32_t* row = a.table + (uint64_t)b * a.table_ld;
    for (int64_t t = lo; t < hi; ++t)
      for (uint32_t h = 0; h < a.hq; ++h) {
        const int64_t pos = kv - (hi - lo) + (t - lo);  // keys 0 .. pos are seen
        const uint16_t* q = a.q + t * a.q_stride + h * a.q_head_stride;
        uint16_t* dst = a.out + t * a.out_stride + (uint64_t)h * a.hd;
        std::fill(o.begin(), o.end(), 0.0);
        double m = -INFINITY, l = 0;
        bool bad = kv > cap;  // the table does not reach that far
        if (!bad) {
          sc.assign(std::max<int64_t>(pos + 1, 0), 0.0);
          for (int64_t k = 0; k <= pos; ++k) {
            const int32_t page = row[k >> a.page_shift];
            if (page < 0 || (uint32_t)page >= a.num_pages) {
              bad = true;
              break;
            }
            const uint16_t* kr = a.pages + page * a.page_stride + (h / g) * a.head_stride + (k & (P - 1)) * a.hd;
            double s = 0;
            for (uint32_t d = 0; d < a.hd; ++d) s += (double)load16(q[d], a.elem) * load16(kr[d], a.elem);
            sc[k] = s * a.scale;
            m = std::max(m, sc[k]);  // a NaN score passes by here and makes the sum NaN
          }
        }
        if (!bad)
          for (int64_t k = 0; k <= pos; ++k) {
            const double p = std::exp(sc[k] - m);
            const uint16_t* vr = a.pages + a.kv_stride + row[k >> a.page_shift] * a.page_stride +
                                 (h / g) * a.head_stride + (k & (P - 1)) * a.hd;
            l += p;
            for (uint32_t d = 0; d < a.hd; ++d) o[d] += p * load16(vr[d], a.elem);
          }
        for (uint32_t d = 0; d < a.hd; ++d)
          dst[d] = store16(bad ? NAN : pos < 0 ? 0.f : (float)(o[d] / l), a.elem);
      }
  }
}

static inline double prob(const void* p, uint64_t i, uint32_t elem) {
  if (elem == ELEM_F32) return reinterpret_cast<const float*>(p)[i];
  return load16(reinterpret_cast<const uint16_t*>(p)[i], elem);
}

void verify_draft_cpu(const VerifyArgs& a) {
  std::vector<double> w(a.V);
  for (uint32_t b = 0; b < a.B; ++b) {
    const uint32_t count = a.counts ? (uint32_t)std::min<int64_t>(std::max(a.counts[b], 0), a.K) : a.K;
    const uint64_t pb = b * a.p_batch, qb = b * a.q_batch;
    uint32_t m = 0;
    for (; m < count; ++m) {
      const int32_t x = a.tokens[(uint64_t)b * a.K + m];
      if (x < 0 || (uint32_t)x >= a.V) break;
      const double qt = a.q ? prob(a.q, qb + m * a.q_row + x, a.elem) : 1.0;
      if (!((double)a.u[(uint64_t)b * a.K + m] * qt < prob(a.p, pb + m * a.p_row + x, a.elem))) break;
    }
    double total = 0, whole = 0;
    for (uint32_t i = 0; i < a.V; ++i) {
      const double p = prob(a.p, pb + m * a.p_row + i, a.elem);
      double q = 0;
      if (m < count)
        q = a.q ? prob(a.q, qb + m * a.q_row + i, a.elem)
                : (int32_t)i == a.tokens[(uint64_t)b * a.K + m] ? 1.0 : 0.0;
      w[i] = p > q && p > 0 ? p - std::max(q, 0.0) : 0.0;
      total += w[i];
      whole += p > 0 ? p : 0.0;
    }
    if (!(total > 0)) {
      total = whole;
      for (uint32_t i = 0; i < a.V; ++i) {
        const double p = prob(a.p, pb + m * a.p_row + i, a.elem);
        w[i] = p > 0 ? p : 0.0;
      }
    }
    const double aim = (double)a.u_last[b] * total;
    double c = 0;
    int32_t pick = -1;
    for (uint32_t i = 0; i < a.V; ++i) {
      c += w[i];
      if (w[i] > 0) pick = (int32_t)i;
      if (w[i] > 0 && c > aim) break;
    }
    int32_t* out = a.out + (uint64_t)b * (a.K + 1);
    for (uint32_t j = 0; j <= a.K; ++j) out[j] = j < m ? a.tokens[(uint64_t)b * a.K + j] : j == m ? pick : -1;
    a.accepted[b] = (int32_t)m;
  }
}

}  // namespace ogkm
