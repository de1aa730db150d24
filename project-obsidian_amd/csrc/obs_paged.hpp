// obs_paged.hpp — what the operators on a paged key/value cache share: the
// checks of their arguments, the sequences as a kernel sees them, and the
// plan that splits their work over workgroups.
#pragma once

#include <algorithm>

#include "obs_internal.hpp"

namespace obs {

// Word of obs_ctx::status_dev (behind the one-launch FFN's): a page id, length,
// entry past the positions or slot out of range that a kernel met.
constexpr uint32_t CTX_ST_PAGED = 2;
static_assert(CTX_ST_PAGED > CTX_ST_FFN_SCHED && CTX_ST_PAGED < CTX_ST_WORDS, "a word of its own");
int paged_status(obs_ctx* ctx);  // reads and clears it (obs_device_status)

constexpr uint32_t PAGED_MAX_SEQS = 4096;
constexpr uint64_t PAGED_MAX_ENTRIES = 1ull << 30;

// Positions of the RoPE table that a call with rope_len builds: a power of two, 8,192
// at least. Tables are built with a wait and kept (graphs read them), so a caller
// whose rope_len follows its longest sequence must not get one a step.
constexpr uint32_t ROPE_ROWS_MIN = 8192;
// From here on the table's angles are formed in double: the fp32 product of
// obs_attn_prep_rows is off by up to 2^-24 of the angle twice, 0.0003 at 8,192, but
// 0.004 at 100,000 and 0.035 at 10^6, beside bf16's half step of 0.002.
constexpr uint32_t ROPE_EXACT_FROM = 8192;
inline uint32_t rope_rows(uint32_t rope_len) {
  uint32_t n = ROPE_ROWS_MIN;
  while (n < rope_len) n *= 2u;  // rope_len <= 2^24
  return n;
}

// Makes the context's device current for a call's launches (a caller may work
// on another one).
struct DeviceGuard {
  int before = -1;
  explicit DeviceGuard(const obs_ctx* ctx) {
    int d = -1;
    if (hipGetDevice(&d) == hipSuccess && d != ctx->device && hipSetDevice(ctx->device) == hipSuccess) before = d;
  }
  ~DeviceGuard() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// Shapes and pointers of kv and seqs; `pointers` false: sizes only.
int check_paged(obs_ctx* ctx, const char* who, const obs_paged_kv* kv, const obs_paged_seqs* seqs, bool pointers);
int check_heads(obs_ctx* ctx, const char* who, uint32_t n_heads, uint32_t n_kv);
int check_grid(obs_ctx* ctx, const char* who, uint64_t workgroups, uint32_t threads);  // a launch holds less than 2^32 threads
int check_weight(obs_ctx* ctx, const char* who, const obs_kv_weight* w, uint64_t entries, bool pointers);

// The pool and the sequences as kernels take them.
struct Paged {
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  const int32_t* table;
  const int32_t* len;
  const int32_t* row;
  uint32_t* status;
  uint32_t n_pages, lp, n_kv, n_seqs, max_pages, n_rows;  // page = 1 << lp
};
inline Paged paged_args(const obs_ctx* ctx, const obs_paged_kv* kv, const obs_paged_seqs* s) {
  return Paged{static_cast<const uint8_t*>(kv->k_pages), static_cast<const uint8_t*>(kv->v_pages),
               kv->k_scale, kv->v_scale, s->pages, s->len, s->row, ctx->status_dev + CTX_ST_PAGED,
               kv->n_pages, static_cast<uint32_t>(__builtin_ctz(kv->page)), kv->n_kv, s->n_seqs, s->max_pages, s->n_rows};
}
struct Weight {
  float* w;
  const int32_t* slot;
  uint32_t n_slots, ld;
};
inline Weight weight_args(const obs_kv_weight* w) {
  return w ? Weight{w->w, w->slot, w->n_slots, w->ld} : Weight{nullptr, nullptr, 0u, 0u};
}

// Arguments of the attention kernels.
struct PagedAttn {
  const uint16_t* q;
  uint16_t* out;
  float* ml;      // of each part and column: maximum and sum
  float* part;    // of each part and column: its unnormalised output
  float* scores;  // [sequence][head][vis]: scores in base 2, where the weights are gathered
  uint2* plan;    // decode: of each sequence its first part and its parts a kv head; prefill: of each tile (uint4)
  uint32_t nh, G, window, sinks, q_ld, vis, min_chunk, target, tiles;
  float scale_log2;
};
// Blocks of 32 that a token can see of a sequence of `entries`.
inline uint64_t most_blocks(uint64_t entries, uint64_t window, uint32_t sinks) {
  const uint64_t all = (entries + 31u) / 32u;
  if (!window) return all;
  const uint64_t w = (window + 31u) / 32u + 1u + (std::min<uint64_t>(sinks, entries) + 31u) / 32u;
  return std::min(all, w);
}
inline size_t up256(size_t n) { return (n + 255u) & ~size_t(255); }
// q, out, weight and the workspace of an attention call; q_ld 0 becomes the dense stride.
int check_attn(obs_ctx* ctx, const char* who, const obs_paged_kv* kv, const obs_paged_seqs* seqs,
               const obs_kv_weight* weight, const uint16_t* q, const uint16_t* out, uint32_t n_heads, uint32_t* q_ld,
               const void* ws, size_t ws_bytes, size_t need);
// Workspace of obs_sdpa_paged_prefill.
size_t prefill_paged_ws(const obs_paged_kv* kv, const obs_paged_seqs* s, uint32_t n_heads, uint32_t window, uint32_t sinks);

}  // namespace obs

namespace obsd {

constexpr float NEG_INF = -__builtin_huge_valf();

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_v;
typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_v;
typedef uint32_t u32x2_v __attribute__((ext_vector_type(2)));

// Reports an argument in device memory that is out of range. The word is only
// ever set to 1, so the order of several stores does not matter.
__device__ __forceinline__ void paged_flag(uint32_t* status) {
  __hip_atomic_store(status, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The functions below that decide what is read are host functions too, so they
// can be tested without a GPU.
__host__ __device__ __forceinline__ uint32_t umin(uint32_t x, uint32_t y) { return x < y ? x : y; }

// Entries of sequence b, within [0, max_pages * page].
__host__ __device__ __forceinline__ uint32_t paged_len(const obs::Paged& a, uint32_t b) {
  const int32_t n = a.len[b];
  const uint32_t cap = a.max_pages << a.lp;
  return n <= 0 ? 0u : umin(static_cast<uint32_t>(n), cap);
}
__host__ __device__ __forceinline__ bool paged_len_bad(const obs::Paged& a, uint32_t b) {
  const int32_t n = a.len[b];
  return n > 0 && static_cast<uint32_t>(n) > (a.max_pages << a.lp);
}
// Token rows [r0, r1) of sequence b, within [0, n_rows].
struct RowSpan {
  uint32_t r0, r1;
};
__host__ __device__ __forceinline__ RowSpan paged_rows(const obs::Paged& a, uint32_t b) {
  if (!a.row) return {b, b + 1u};
  const int32_t lo = a.row[b], hi = a.row[b + 1u];
  const uint32_t r0 = umin(lo > 0 ? static_cast<uint32_t>(lo) : 0u, a.n_rows);
  const uint32_t r1 = umin(hi > 0 ? static_cast<uint32_t>(hi) : 0u, a.n_rows);
  return {r0, r1 > r0 ? r1 : r0};
}

// Page id of entry j; `ok` is false for an id out of range, which then reads as page 0.
__host__ __device__ __forceinline__ uint32_t paged_id(const obs::Paged& a, uint32_t b, uint32_t j, bool& ok) {
  const uint32_t id = static_cast<uint32_t>(a.table[static_cast<size_t>(b) * a.max_pages + umin(j >> a.lp, a.max_pages - 1u)]);
  ok = id < a.n_pages;
  return ok ? id : 0u;
}

// What a query sees, in blocks of 32 entries.
// Entry j of the queries at entries i0 <= i <= i1: the blocks that hold the
// first `sinks` entries and those from the window of i0 to i1. Block x of the
// nblk listed ones starts at entry 32 * (x < sb ? x : x - sb + wb).
struct Span {
  uint32_t hi, lo, sb, wb, nblk;
  __host__ __device__ __forceinline__ uint32_t start(uint32_t x) const { return 32u * (x < sb ? x : x - sb + wb); }
};
__host__ __device__ __forceinline__ Span span_of(uint32_t i0, uint32_t hi, uint32_t window, uint32_t sinks) {
  Span s;
  s.hi = hi;
  s.lo = window && i0 + 1u > window ? i0 + 1u - window : 0u;
  s.wb = s.lo / 32u;
  s.sb = umin((umin(sinks, hi) + 31u) / 32u, s.wb);
  s.nblk = hi ? s.sb + (hi + 31u) / 32u - s.wb : 0u;
  return s;
}

// Slot of sequence b's gathered weight, or -1.
__device__ __forceinline__ int64_t weight_slot(const obs::Weight& w, uint32_t b) {
  const int32_t s = w.slot ? w.slot[b] : static_cast<int32_t>(b);
  return s >= 0 && static_cast<uint32_t>(s) < w.n_slots ? static_cast<int64_t>(s) : -1;
}

// fp32 pair -> two e4m3 bytes (OCP, round to nearest even; beyond 448 -> 448, NaN stays NaN).
__device__ __forceinline__ float e4m3_clamp(float v) {
  return v != v ? v : __builtin_fminf(__builtin_fmaxf(v, -448.0f), 448.0f);
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(a), e4m3_clamp(b), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(c), e4m3_clamp(d), r, true);
  return static_cast<uint32_t>(r);
}
// Two e4m3 bytes (the low or the high half of w) -> two bf16, exact (3 mantissa bits).
template <bool HIGH>
__device__ __forceinline__ uint32_t e4m3x2_bf16(uint32_t w) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
}

// The entries of the block of 32 from entry t that are below hi, and at or above
// lo or below sinks: a bit each. Arithmetic on whole words, no branch an entry.
__host__ __device__ __forceinline__ uint32_t below_bits(uint32_t t, uint32_t end) {  // entries below `end`
  const uint32_t n = end > t ? umin(end - t, 32u) : 0u;
  return n == 32u ? ~0u : (1u << n) - 1u;
}
__host__ __device__ __forceinline__ uint32_t seen_bits(uint32_t t, uint32_t hi, uint32_t lo, uint32_t sinks) {
  return below_bits(t, hi) & (~below_bits(t, lo) | below_bits(t, sinks));
}
// Word masks of eight bf16 from their bits 0 .. 7.
__device__ __forceinline__ u32x4_v word_masks(uint32_t bits) {
  u32x4_v m;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t a = static_cast<uint32_t>(static_cast<int32_t>(bits << (31u - 2u * i)) >> 31);
    const uint32_t b = static_cast<uint32_t>(static_cast<int32_t>(bits << (30u - 2u * i)) >> 31);
    m[i] = (a & 0xffffu) | (b & 0xffff0000u);
  }
  return m;
}

// Sum and inclusive scan over a wave by DPP (rows of 16 lanes, then the row
// broadcasts): a few VALU steps instead of six trips through the LDS crossbar.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_add(uint32_t v) {
  return v + static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {  // inclusive
  v = dpp_add<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  v = dpp_add<DPP_ROW_BCAST15, 0xA>(v);
  return dpp_add<DPP_ROW_BCAST31, 0xC>(v);
}
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {  // uniform
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(wave_scan_u32(v)), 63));
}
__device__ __forceinline__ float wave_max_f32(float v) {  // uniform
  v = fmaxf(v, dpp_f32<DPP_XOR1>(v));
  v = fmaxf(v, dpp_f32<DPP_XOR2>(v));
  v = fmaxf(v, dpp_f32<DPP_HALF_MIRROR>(v));
  v = fmaxf(v, dpp_f32<DPP_MIRROR>(v));
  return fmaxf(fmaxf(readlane_f32(v, 0), readlane_f32(v, 16)), fmaxf(readlane_f32(v, 32), readlane_f32(v, 48)));
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
}
// Parts of a sequence's nblk blocks.
__device__ __forceinline__ uint32_t plan_splits(uint32_t nblk, uint32_t chunk) { return max(1u, (nblk + chunk - 1u) / chunk); }

}  // namespace obsd
