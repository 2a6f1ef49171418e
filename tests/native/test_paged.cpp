// CPU references of the paged-serving ops (csrc/core/paged_ref.cpp) on heap buffers of
// exactly the size the ops may touch, built with g++ under AddressSanitizer + UBSan and
// run by tests/test_native_paged.py: the contents here are those that steer an index
// (lengths, page ids, slots, tokens), at and beyond their limits.
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <memory>
#include <vector>

#include "ogkm/paged.hpp"

using namespace ogkm;

static int g_fail = 0;
#define CHECK(c)                                                           \
  do {                                                                     \
    if (!(c)) {                                                            \
      fprintf(stderr, "CHECK failed %s:%d: %s\n", __FILE__, __LINE__, #c); \
      g_fail++;                                                            \
    }                                                                      \
  } while (0)

typedef std::vector<int32_t> Ints;
static const uint16_t kOne = 0x3F80, kNan = 0x7FC0;  // bf16

struct Planned {
  Ints cu, kv, counts, granted, pos, slots, start, table;
};
static Planned plan(const Ints& fresh, const Ints& kv, const Ints& held, Ints table, uint32_t width, uint32_t ld,
                    const Ints& free_pages, int32_t start, uint32_t n) {
  const uint32_t B = (uint32_t)fresh.size();
  Planned r{Ints(B + 1), Ints(B), Ints(B), Ints(B), Ints(n), Ints(n), Ints(1), table};
  PlanArgs a{fresh.data(), kv.data(),       held.data(), r.table.data(), free_pages.data(), &start,
             r.cu.data(),  r.kv.data(),     r.counts.data(), r.granted.data(), r.pos.data(), r.slots.data(),
             r.start.data(), ld, B, width, (uint32_t)free_pages.size(), 4, n};
  paged_plan_cpu(a);
  return r;
}

static void test_plan() {
  // the free list runs out: one page of two for the first, three wanted by the second
  Planned p = plan({16, 33, 1}, {0, 0, 15}, {0, 0, 1}, Ints(9, -1), 3, 3, {7, 8}, 0, 50);
  CHECK((p.granted == Ints{1, 0, 1}) && p.start[0] == 1 && p.table[0] == 7 && p.slots[0] == 7 * 16 && p.slots[16] == -1);
  CHECK(p.slots[49] == -1 && p.pos[49] == 15);  // a held page that is none
  // an empty free list, and one whose start lies behind its end or before its begin
  p = plan({1, 1}, {15, 16}, {1, 1}, Ints{4, -1, 5, -1}, 2, 2, {}, 0, 2);
  CHECK((p.granted == Ints{1, 0}) && p.slots[0] == 4 * 16 + 15 && p.slots[1] == -1);
  p = plan({1}, {0}, {0}, Ints(1, -1), 1, 1, {3}, 9, 1);
  CHECK(p.granted[0] == 0 && p.start[0] == 1);
  p = plan({1}, {0}, {0}, Ints(1, -1), 1, 1, {3}, INT_MIN, 1);
  CHECK(p.granted[0] == 1 && p.slots[0] == 48 && p.start[0] == 1);
  // a table row filled to its end, one too short by a token, rows apart by more than the width
  p = plan({32, 33}, {0, 0}, {0, 0}, Ints(3 + 2, -1), 2, 3, {0, 1, 2, 3, 4, 5}, 0, 65);
  CHECK((p.granted == Ints{1, 0}) && p.slots[31] == 31 && p.slots[32] == -1 && p.table[1] == 1 && p.table[3] == -1);
  // more rows than the batch; the largest lengths, counts beyond the table, negative ones
  p = plan({4, 4}, {0, 0}, {1, 1}, Ints(2, 0), 1, 1, {1}, 0, 7);
  CHECK((p.granted == Ints{1, 0}) && (p.cu == Ints{0, 4, 7}));
  p = plan({INT_MAX, INT_MAX, 1}, {INT_MAX, 0, INT_MAX}, {0, INT_MAX, INT_MAX}, Ints(3, 0), 1, 1, {1}, 0, 1);
  CHECK((p.granted == Ints{0, 0, 0}) && p.pos[0] == -1 && (p.counts == Ints{0, 1, 1}));
  p = plan({INT_MIN, 1}, {INT_MIN, -1}, {INT_MIN, -5}, Ints(2, 9), 1, 1, {6}, 0, 1);
  CHECK((p.granted == Ints{1, 1}) && p.slots[0] == 6 * 16 && p.table[0] == 9);
  // page ids whose slots do not fit 32 bits
  p = plan({1, 1, 1}, {0, 0, 0}, {1, 1, 1}, Ints{INT_MAX, INT_MIN, INT_MAX >> 4}, 1, 1, {}, 0, 3);
  CHECK((p.granted == Ints{1, 1, 1}) && p.slots[0] == -1 && p.slots[1] == -1 && p.slots[2] == (INT_MAX >> 4) * 16);
  // nobody
  p = plan({}, {}, {}, {}, 1, 1, {1}, 0, 3);
  CHECK(p.cu[0] == 0 && p.pos[2] == -1 && p.start[0] == 0);
  p = plan({0}, {5}, {1}, Ints(1, 2), 1, 1, {}, 0, 0);
  CHECK(p.granted[0] == 1 && p.kv[0] == 5);
}

static void test_rope() {
  const uint32_t hq = 2, hkv = 1, hd = 16, P = 16, num = 2, max_pos = 3;
  const std::vector<int32_t> pos{0, 2, 3, -1, INT_MAX, 1, 1, 1}, slots{0, 31, 5, 6, 7, 32, -1, INT_MAX};
  const uint32_t n = (uint32_t)pos.size();
  std::vector<uint16_t> qkv(n * (hq + 2 * hkv) * hd, kOne), q(n * hq * hd), pages(2 * num * hkv * P * hd, kNan);
  std::vector<float> cos(max_pos * hd / 2, 1.f), sin(max_pos * hd / 2, 0.f);
  PagedRopeArgs a{qkv.data(), (hq + 2 * hkv) * hd, cos.data(), sin.data(), pos.data(), slots.data(), q.data(),
                  pages.data(), num * hkv * P * hd, hkv * P * hd, P * hd, n, hq, hkv, hd, num, 4, max_pos, ELEM_BF16};
  paged_rope_cpu(a);
  auto k = [&](uint32_t slot) { return pages[slot * hd]; };
  auto v = [&](uint32_t slot) { return pages[(num * P + slot) * hd]; };
  CHECK(k(0) == kOne && v(0) == kOne && k(31) == kOne && v(31) == kOne);
  CHECK((k(5) & 0x7FFF) > 0x7F80 && v(5) == kOne);      // a position behind the tables: k is NaN, v as it is
  CHECK(k(6) == kNan && v(6) == kNan && q[3 * hq * hd] == 0);  // a row of padding
  CHECK((q[4 * hq * hd] & 0x7FFF) > 0x7F80 && q[7 * hq * hd] == kOne);
  CHECK(v(1) == kNan && v(30) == kNan);
}

struct Attn {
  uint32_t n, hq = 2, hkv = 1, hd = 64, num = 3, width = 2;
  std::vector<uint16_t> q, pages, out;
  explicit Attn(uint32_t rows) : n(rows), q(rows * hq * hd, kOne), pages(2 * num * hkv * 16 * hd, kOne), out(rows * hq * hd, 7) {}
  void run(const Ints& cu, const Ints& kv, const Ints& table, uint32_t elem = ELEM_BF16) {
    PagedAttnArgs a{};
    a.q = q.data();
    a.q_stride = hq * hd;
    a.q_head_stride = hd;
    a.pages = pages.data();
    a.kv_stride = num * hkv * 16 * hd;
    a.page_stride = hkv * 16 * hd;
    a.head_stride = 16 * hd;
    a.cu_q = cu.data();
    a.kv_lens = kv.data();
    a.table = table.data();
    a.table_ld = width;
    a.out = out.data();
    a.out_stride = hq * hd;
    a.n = n;
    a.B = (uint32_t)kv.size();
    a.hq = hq;
    a.hkv = hkv;
    a.hd = hd;
    a.num_pages = num;
    a.page_shift = 4;
    a.width = width;
    a.scale = 0.125f;
    a.elem = elem;
    paged_attn_cpu(a);
  }
  uint16_t at(uint32_t row) const { return out[row * hq * hd]; }
  bool nan(uint32_t row) const { return (at(row) & 0x7FFF) > 0x7F80; }
};

static void test_attention() {
  Attn x(4);
  x.run({0, 1, 2, 3, 4}, {32, 33, INT_MAX, -3}, {0, 2, 0, 1, 1, 0, 0, 0});
  CHECK(x.at(0) == kOne && x.nan(1) && x.nan(2) && x.at(3) == 0);  // a full table row, longer ones, no token
  Attn y(4);
  y.run({0, 1, 2, 3, 4}, {17, 17, 16, 17}, {0, 3, INT_MIN, 1, 2, INT_MAX, INT_MAX, 0});
  CHECK(y.nan(0) && y.nan(1) && y.at(2) == kOne && y.nan(3));  // pages outside the pool, one of them not needed
  Attn z(5);  // more rows than keys; bounds outside q; falling bounds
  z.run({INT_MIN, 3, 1, INT_MAX}, {1, 0, 2}, {0, 0, 0, 0, 1, 1});
  CHECK(z.at(0) == 0 && z.at(3) == kOne && z.at(4) == kOne);
  Attn w(2);  // no request, and none with rows
  w.run({0}, {}, {});
  w.run({2, 2}, {5}, {0, 0});
  CHECK(w.at(0) == 7 && w.at(1) == 7);
  Attn f(1);  // every fp16 bit pattern as a value
  for (uint32_t v = 0; v < 65536; v += 64) {
    for (uint32_t d = 0; d < 64; ++d) f.pages[f.num * 16 * f.hd + d] = (uint16_t)(v + d);
    for (auto& k : f.q) k = 0x3C00;
    for (uint32_t d = 0; d < 64; ++d) f.pages[d] = 0;
    f.run({0, 1}, {1}, {0, 0}, ELEM_F16);
    for (uint32_t d = 0; d < 64; ++d) {
      const uint16_t in = (uint16_t)(v + d), got = f.out[d];
      CHECK((in & 0x7FFF) > 0x7C00 ? (got & 0x7FFF) > 0x7C00 : got == in || (!(in & 0x7FFF) && !(got & 0x7FFF)));
    }
  }
}

struct Verified {
  Ints out, accepted;
};
static Verified verify(const std::vector<float>& p, const std::vector<float>* q, const Ints& tokens,
                       const std::vector<float>& u, const std::vector<float>& last, const Ints* counts, uint32_t K,
                       uint32_t V) {
  const uint32_t B = (uint32_t)last.size();
  Verified r{Ints(B * (K + 1)), Ints(B)};
  VerifyArgs a{p.data(), (uint64_t)(K + 1) * V, V, q ? q->data() : nullptr, (uint64_t)K * V, V, tokens.data(), u.data(),
               last.data(), counts ? counts->data() : nullptr, r.out.data(), r.accepted.data(), nullptr, B, K, V, ELEM_F32};
  verify_draft_cpu(a);
  return r;
}

static void test_verify() {
  const Ints many{INT_MAX, INT_MIN};
  // a vocabulary of one entry, no drafts
  Verified r = verify({1.f, 0.f}, nullptr, {}, {}, {0.5f, 0.f}, &many, 0, 1);
  CHECK((r.out == Ints{0, -1}) && (r.accepted == Ints{0, 0}));
  // tokens outside the vocabulary, at both ends
  const std::vector<float> p{.5f, .5f, 1.f, 0.f, .5f, .5f, 0.f, 1.f, 0.f, 1.f, 1.f, 0.f, 0.f, 1.f, 1.f, 0.f};
  const std::vector<float> q(8, .5f);
  r = verify(p, &q, {2, -1, INT_MIN, INT_MAX}, {0.f, 0.f, 0.f, 0.f}, {0.f, .9f}, nullptr, 1, 2);
  CHECK((r.accepted == Ints{0, 0}));
  r = verify({0.f, 1.f, 1.f, 0.f, 0.f, 1.f, 1.f, 0.f}, nullptr, {1, 0}, {.5f, .5f}, {.5f, .5f}, &many, 1, 2);
  CHECK((r.accepted == Ints{1, 0}) && (r.out == Ints{1, 0, 1, -1}));
  // all weight gone, NaN
  r = verify({NAN, -1.f, 0.f, NAN}, nullptr, {0}, {.5f}, {NAN}, nullptr, 1, 2);
  CHECK((r.accepted == Ints{0}) && (r.out == Ints{-1, -1}));
}

int main() {
  test_plan();
  test_rope();
  test_attention();
  test_verify();
  if (g_fail) {
    fprintf(stderr, "%d check(s) failed\n", g_fail);
    return 1;
  }
  fprintf(stderr, "ALL NATIVE TESTS PASSED\n");
  return 0;
}
