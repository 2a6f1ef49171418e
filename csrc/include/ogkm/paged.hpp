// Serving ops over a paged KV cache and speculative decoding: argument structs
// shared by the HIP kernels (csrc/kernels/paged_*.hip, speculative.hip), the
// CPU references of the fake backend (csrc/core/paged_ref.cpp) and the bindings.
//
// Page pool: [2][num_pages][hkv][P][hd] (k then v) - the contiguous cache's
// [2][B][hkv][T][hd] with pages in place of sequences, so a (page, kv head) is
// one contiguous run of P rows. The three outer strides are free. A block table
// row lists the pages of one request: token t lies in page table[t / P], row t % P.
#pragma once

#include <cstdint>

namespace ogkm {

enum ElemType : uint32_t { ELEM_BF16 = 0, ELEM_F16 = 1, ELEM_F32 = 2 };

constexpr uint32_t kPlanMaxRequests = 4096;  // the per-request state of the scan stays in LDS (9 B each)

// One step of a batch: where every new token goes. All lengths live in device
// memory; nothing is read back. page_size is a power of two.
struct PlanArgs {
  const int32_t* new_lens;     // [B] tokens this step appends to each request
  const int32_t* kv_lens;      // [B] tokens already cached
  const int32_t* page_counts;  // [B] pages a request holds
  int32_t* table;              // [B][table_ld], new pages are written behind the held ones
  const int32_t* free_pages;   // [n_free]
  const int32_t* free_start;   // [1] first unused entry of free_pages
  int32_t* cu_q;               // [B + 1]
  int32_t* kv_out;             // [B]
  int32_t* counts_out;         // [B]
  int32_t* granted;            // [B]
  int32_t* positions;          // [n_tokens]
  int32_t* slots;              // [n_tokens]
  int32_t* free_out;           // [1]
  uint64_t table_ld;
  uint32_t B, width, n_free, page_shift, n_tokens;
};

struct PagedRopeArgs {
  const uint16_t* qkv;       // [n, (hq + 2 hkv) hd], row stride ldqkv
  uint64_t ldqkv;
  const float* cos;          // [max_pos, hd / 2]
  const float* sin;
  const int32_t* positions;  // [n]
  const int32_t* slots;      // [n]
  uint16_t* q_out;           // [n, hq, hd]
  uint16_t* pages;
  uint64_t kv_stride, page_stride, head_stride;  // elements
  uint32_t n, hq, hkv, hd, num_pages, page_shift, max_pos;
  uint32_t elem;             // ELEM_BF16 / ELEM_F16
};

// How a call's work is laid out: from the host's bounds alone, so that one layout
// serves every content of the device's lengths.
struct PagedAttnPlan {
  uint32_t most_rows;   // rows of a request per kv head, by the host's bound
  uint32_t few_rows;    // requests of up to so many rows per kv head take the `few` body
  uint32_t few_blocks;  // its column blocks of 16 rows: 1 or 2
  uint32_t few_waves;   // waves of a workgroup: 4 or 8
  uint32_t few_splits;  // its splits of the key axis, at most
  uint32_t many_tiles;  // 128-row tiles of the other requests, at most (0: none expected)
  uint32_t many_splits;
  uint32_t many_sorted; // 1: tiles in the order of their requests' keys (B <= 64)
  uint64_t few_part;    // rows of partial results of the few-row requests,
  uint64_t part_rows;   // and of all (hd + 2 floats each)
};
PagedAttnPlan paged_attn_plan(uint32_t n, uint32_t B, uint32_t hq, uint32_t hkv, uint32_t hd, uint32_t max_q,
                              uint32_t max_kv);

struct PagedAttnArgs {
  const uint16_t* q;         // [n, hq, hd]; strides of a row and of a head
  uint64_t q_stride, q_head_stride;
  const uint16_t* pages;
  uint64_t kv_stride, page_stride, head_stride;
  const int32_t* cu_q;       // [B + 1]
  const int32_t* kv_lens;    // [B] including the new tokens
  const int32_t* table;      // [B][table_ld]
  uint64_t table_ld;
  uint16_t* out;             // [n, hq * hd], row stride out_stride
  uint64_t out_stride;
  uint32_t n, B, hq, hkv, hd, num_pages, page_shift, width;
  float scale;
  uint32_t elem;
  PagedAttnPlan plan;        // GPU: how the work is split, and the splits' partial results
  float* part_o;
  float* part_ml;
};

struct VerifyArgs {
  const void* p;             // [B, K + 1, V] target probabilities; strides of the first two dims
  uint64_t p_batch, p_row;
  const void* q;             // [B, K, V] draft probabilities, or null: drafts were certain
  uint64_t q_batch, q_row;
  const int32_t* tokens;     // [B, K] drafted
  const float* u;            // [B, K] uniform numbers of the acceptance tests
  const float* u_last;       // [B] uniform numbers of the last token
  const int32_t* counts;     // [B] drafts of each request, or null: K
  int32_t* out;              // [B, K + 1], -1 behind the last token
  int32_t* accepted;         // [B]
  double* sums;              // [B, ceil(V / kVerifyChunk)] residual of each chunk
  uint32_t B, K, V, elem;
};
constexpr uint32_t kVerifyChunk = 4096;  // vocabulary entries of one partial sum

// CPU references (fake backend, tests).
void paged_plan_cpu(const PlanArgs& a);
void paged_rope_cpu(const PagedRopeArgs& a);
void paged_attn_cpu(const PagedAttnArgs& a);
void verify_draft_cpu(const VerifyArgs& a);

}  // namespace ogkm
