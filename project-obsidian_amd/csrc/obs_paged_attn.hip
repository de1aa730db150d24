// obs_paged_attn.hip — attention over a paged key/value cache: one new token of
// every sequence (obs_sdpa_paged_decode) and the token rows of a batch of
// prompts (obs_sdpa_paged_prefill), with a sliding window that keeps the first
// tokens visible.
#include <algorithm>

#include "obs_paged.hpp"

namespace {
using namespace obsd;
using obs::Paged;
using obs::Weight;

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float f32x4_v;

constexpr float NEG_INF = -__builtin_huge_valf();

struct AttnArgs {
  const uint16_t* q;
  uint16_t* out;
  float* ml;      // [item][16][2]: maximum and sum of a part
  float* part;    // [item][G][HD]: its unnormalised output
  float* scores;  // [sequence][head][vis]: scores in base 2, where the weights are gathered
  uint32_t nh, G, window, sinks, q_ld, vis, min_chunk, target;
  float scale_log2;
};

// ---------------------------------------------------------------------------
// One block of 32 entries for one wave: 16 columns of queries
// ---------------------------------------------------------------------------
// S^T [32 entries x 16 columns] = K . Q^T by two v_mfma_f32_16x16x32_bf16 per 32
// dims, then O^T [dims x 16 columns] += V^T . P. A lane (col = lane % 16, g =
// lane / 16) ends with column col throughout, so every factor of the softmax is
// its own. Row r of score tile tt is entry 8 (r / 4) + 4 tt + r % 4 of the block:
// the lane's eight scores are then entries 8 g .. 8 g + 7, the eight values that
// one 16-byte load of a transposed value row brings.
template <uint32_t HD, bool F8>
struct Block {
  static constexpr uint32_t KS = HD / 32u, NT = HD / 16u, KL = F8 ? KS / 2u : KS;
  u32x4_v k[2][KL];  // e4m3: 16 dims a load, two steps
  typename std::conditional<F8, u32x2_v, u32x4_v>::type v[NT];

  // kp, vp: page ids of the lane's key rows and values; t0: first entry
  __device__ __forceinline__ void load(const Paged& a, uint32_t kv, uint32_t kp, uint32_t vp, uint32_t t0, uint32_t col,
                                       uint32_t g) {
    const uint32_t mask = (1u << a.lp) - 1u;
    constexpr uint32_t SZ = F8 ? 1u : 2u;
    const uint8_t* kb = a.k + ((static_cast<size_t>(kp) * a.n_kv + kv) << a.lp) * (HD * SZ);
    const uint8_t* vb = a.v + ((static_cast<size_t>(vp) * a.n_kv + kv) * HD << a.lp) * SZ + ((t0 + 8u * g) & mask) * SZ;
#pragma unroll
    for (uint32_t tt = 0; tt < 2; ++tt) {
      const uint8_t* kr = kb + ((t0 + 8u * (col / 4u) + 4u * tt + col % 4u) & mask) * (HD * SZ) + 16u * g;
#pragma unroll
      for (uint32_t i = 0; i < KL; ++i) k[tt][i] = *reinterpret_cast<const u32x4_v*>(kr + 64u * i);
    }
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt) {
      const uint8_t* vr = vb + ((16u * nt + col) * SZ << a.lp);
      if constexpr (F8)
        v[nt] = *reinterpret_cast<const u32x2_v*>(vr);
      else
        v[nt] = *reinterpret_cast<const u32x4_v*>(vr);
    }
  }
  // key fragment of tile tt, step ks: the dims that query fragment ks holds
  __device__ __forceinline__ bf16x8_v key(uint32_t tt, uint32_t ks) const {
    if constexpr (F8) {
      const u32x4_v x = k[tt][ks / 2u];
      const uint32_t w0 = ks & 1u ? x.z : x.x, w1 = ks & 1u ? x.w : x.y;
      return __builtin_bit_cast(bf16x8_v, u32x4_v{e4m3x2_bf16<false>(w0), e4m3x2_bf16<true>(w0), e4m3x2_bf16<false>(w1),
                                                  e4m3x2_bf16<true>(w1)});
    } else {
      return __builtin_bit_cast(bf16x8_v, k[tt][ks]);
    }
  }
  __device__ __forceinline__ u32x4_v value(uint32_t nt) const {
    if constexpr (F8)
      return u32x4_v{e4m3x2_bf16<false>(v[nt].x), e4m3x2_bf16<true>(v[nt].x), e4m3x2_bf16<false>(v[nt].y),
                     e4m3x2_bf16<true>(v[nt].y)};
    else
      return v[nt];
  }
  // dims of query fragment ks: 32 ks + 8 g in bf16; 64 (ks / 2) + 16 g + 8 (ks % 2) in e4m3
  static __device__ __forceinline__ uint32_t q_dim(uint32_t ks, uint32_t g) {
    return F8 ? 64u * (ks / 2u) + 16u * g + 8u * (ks & 1u) : 32u * ks + 8u * g;
  }
};

// Word masks of eight consecutive bf16 from entry t: those below hi, and at or
// above lo or below sinks, are kept.
__device__ __forceinline__ u32x4_v entry_masks(uint32_t t, uint32_t hi, uint32_t lo, uint32_t sinks, bool ok) {
  u32x4_v m;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t a = t + 2u * i, b = a + 1u;
    const bool sa = ok && a < hi && (a >= lo || a < sinks), sb = ok && b < hi && (b >= lo || b < sinks);
    m[i] = (sa ? 0xffffu : 0u) | (sb ? 0xffff0000u : 0u);
  }
  return m;
}

// Running softmax of a column and its output.
template <uint32_t HD>
struct Column {
  float m = NEG_INF, l = 0.0f;  // l: the lane's share (its own entries)
  f32x4_v o[HD / 16u];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t nt = 0; nt < HD / 16u; ++nt) o[nt] = f32x4_v{0.0f, 0.0f, 0.0f, 0.0f};
  }
};

// One block into the lane's column. hi, lo: the column's own limits; vhi, vlo:
// the limits of what any column of the wave sees (values outside read as zero:
// the pool may hold anything there). masked: whether the block needs any of it.
template <uint32_t HD, bool F8>
__device__ __forceinline__ void block_step(const Block<HD, F8>& blk, const bf16x8_v (&qb)[HD / 32u], Column<HD>& c,
                                           uint32_t t, uint32_t hi, uint32_t lo, uint32_t vhi, uint32_t vlo,
                                           uint32_t sinks, bool ok, bool masked, float scale_log2, float (&sv)[8],
                                           uint32_t lane) {
  constexpr uint32_t KS = HD / 32u, NT = HD / 16u;
#pragma unroll
  for (uint32_t tt = 0; tt < 2; ++tt) {
    f32x4_v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(blk.key(tt, ks), qb[ks], acc, 0, 0, 0);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) sv[4 * tt + i] = acc[i] * scale_log2;
  }
  if (masked) {
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t e = t + j;
      sv[j] = ok && e < hi && (e >= lo || e < sinks) ? sv[j] : NEG_INF;
    }
  }
  float bm = sv[0];
#pragma unroll
  for (uint32_t j = 1; j < 8; ++j) bm = fmaxf(bm, sv[j]);
  bm = fmaxf(bm, lane_xor16_f32(bm, lane));
  bm = fmaxf(bm, lane_xor32_f32(bm, lane));
  const float m_new = fmaxf(c.m, bm), m_use = m_new == NEG_INF ? 0.0f : m_new;
  const float corr = __builtin_amdgcn_exp2f(c.m - m_use);
  float p[8], sum = 0.0f;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    p[j] = __builtin_amdgcn_exp2f(sv[j] - m_use);
    sum += p[j];  // the sum in fp32; P is rounded to bf16 for the product only
  }
  c.l = __builtin_fmaf(c.l, corr, sum);
  c.m = m_new;
  const bf16x8_v pb = __builtin_bit_cast(bf16x8_v, u32x4_v{pack_bf16_pair_rne(p[0], p[1]), pack_bf16_pair_rne(p[2], p[3]),
                                                           pack_bf16_pair_rne(p[4], p[5]), pack_bf16_pair_rne(p[6], p[7])});
  u32x4_v vm = {~0u, ~0u, ~0u, ~0u};
  if (masked) vm = entry_masks(t, vhi, vlo, sinks, ok);
#pragma unroll
  for (uint32_t nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) c.o[nt][i] *= corr;
    const u32x4_v vv = blk.value(nt);
    const bf16x8_v va = __builtin_bit_cast(bf16x8_v, u32x4_v{vv.x & vm.x, vv.y & vm.y, vv.z & vm.z, vv.w & vm.w});
    c.o[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb, c.o[nt], 0, 0, 0);
  }
}

// ---------------------------------------------------------------------------
// The plan: which part of which sequence a workgroup takes
// ---------------------------------------------------------------------------
// Every sequence's blocks are cut into parts of `chunk` blocks, chunk so that
// the call has about `target` parts (and at least min_chunk blocks), by all
// lengths of the call: each wave adds them up itself, 64 sequences at a time.
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) v += static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), k, 64));
  return v;
}
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v, uint32_t lane) {  // inclusive
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const uint32_t o = static_cast<uint32_t>(__shfl_up(static_cast<int>(v), k, 64));
    v += lane >= static_cast<uint32_t>(k) ? o : 0u;
  }
  return v;
}
__device__ __forceinline__ Span decode_span(const Paged& a, const AttnArgs& p, uint32_t b) {
  const uint32_t n = paged_len(a, b);
  return span_of(n ? n - 1u : 0u, n, p.window, p.sinks);
}
__device__ __forceinline__ uint32_t plan_chunk(const Paged& a, const AttnArgs& p, uint32_t lane) {
  uint64_t total = 0;
  for (uint32_t base = 0; base < a.n_seqs; base += 64u) {
    const uint32_t b = base + lane;
    total += wave_sum_u32(b < a.n_seqs ? decode_span(a, p, b).nblk : 0u);
  }
  total *= a.n_kv;
  return max(p.min_chunk, static_cast<uint32_t>((total + p.target - 1u) / p.target));
}
__device__ __forceinline__ uint32_t plan_splits(uint32_t nblk, uint32_t chunk) { return max(1u, (nblk + chunk - 1u) / chunk); }
// Parts of the sequences before b.
__device__ __forceinline__ uint32_t plan_first(const Paged& a, const AttnArgs& p, uint32_t chunk, uint32_t b, uint32_t lane) {
  uint32_t first = 0;
  for (uint32_t base = 0; base < b; base += 64u) {
    const uint32_t o = base + lane;
    first += wave_sum_u32(o < b ? plan_splits(decode_span(a, p, o).nblk, chunk) : 0u);
  }
  return first * a.n_kv;
}
// The sequence of part `item` and its first part; n_seqs behind the last.
struct Found {
  uint32_t b, first;
};
__device__ __forceinline__ Found plan_find(const Paged& a, const AttnArgs& p, uint32_t chunk, uint32_t item, uint32_t lane) {
  uint32_t acc = 0;
  for (uint32_t base = 0; base < a.n_seqs; base += 64u) {
    const uint32_t b = base + lane;
    const uint32_t own = b < a.n_seqs ? a.n_kv * plan_splits(decode_span(a, p, b).nblk, chunk) : 0u;
    const uint32_t incl = wave_scan_u32(own, lane);
    const uint32_t all = __builtin_amdgcn_readlane(incl, 63);
    if (item < acc + all) {
      const uint32_t before = static_cast<uint32_t>(__popcll(__ballot(acc + incl <= item)));
      const uint32_t first = acc + (before ? static_cast<uint32_t>(__builtin_amdgcn_readlane(incl, before - 1u)) : 0u);
      return {base + before, first};
    }
    acc += all;
  }
  return {a.n_seqs, 0u};
}

// ---------------------------------------------------------------------------
// One new token a sequence
// ---------------------------------------------------------------------------
// A workgroup takes one part of one (sequence, kv head); the G query heads are
// the columns. Its four waves take the part's blocks in turn and meet in LDS.
// A part that is all of its sequence writes the output, others their maximum,
// sum and output for paged_join_kernel.
template <uint32_t HD, bool F8, bool WEIGHT>
__global__ void __launch_bounds__(256) paged_decode_kernel(Paged a, AttnArgs p) {
  constexpr uint32_t NT = HD / 16u;
  __shared__ float s_ml[4][16][2];
  __shared__ float s_o[4][16][HD + 4u];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, col = lane & 15u, g = lane >> 4;
  const uint32_t chunk = __builtin_amdgcn_readfirstlane(plan_chunk(a, p, lane));
  const Found f = plan_find(a, p, chunk, blockIdx.x, lane);
  const uint32_t b = __builtin_amdgcn_readfirstlane(f.b);
  if (b >= a.n_seqs) return;  // uniform
  const Span s = decode_span(a, p, b);
  const uint32_t splits = plan_splits(s.nblk, chunk), at = blockIdx.x - __builtin_amdgcn_readfirstlane(f.first);
  const uint32_t kv = at / splits, sp = at % splits;
  const uint32_t x0 = sp * chunk, x1 = min(s.nblk, x0 + chunk);
  if (tid == 0u && at == 0u && paged_len_bad(a, b)) paged_flag(a.status);
  const float scale = F8 ? p.scale_log2 * a.k_scale[kv] : p.scale_log2;
  bf16x8_v qb[HD / 32u];
#pragma unroll
  for (uint32_t ks = 0; ks < HD / 32u; ++ks) {
    u32x4_v v = *reinterpret_cast<const u32x4_v*>(p.q + static_cast<size_t>(b) * p.q_ld + (kv * p.G + min(col, p.G - 1u)) * HD +
                                                  Block<HD, F8>::q_dim(ks, g));
    if (col >= p.G) v = u32x4_v{0u, 0u, 0u, 0u};
    qb[ks] = __builtin_bit_cast(bf16x8_v, v);
  }
  Column<HD> c;
  c.clear();
  // page ids of the wave's next 64 blocks (both halves of each), a block a lane
  uint32_t id0 = 0, id1 = 0;
  for (uint32_t x = x0 + wave, it = 0; x < x1; x += 4u, ++it) {
    if ((it & 63u) == 0u) {
      const uint32_t t = s.start(min(x + 4u * lane, x1 - 1u));
      const size_t row = static_cast<size_t>(b) * a.max_pages;
      id0 = static_cast<uint32_t>(a.table[row + min(t >> a.lp, a.max_pages - 1u)]);
      id1 = static_cast<uint32_t>(a.table[row + min((t + 16u) >> a.lp, a.max_pages - 1u)]);
    }
    const uint32_t t0 = s.start(x);
    uint32_t p0 = __builtin_amdgcn_readlane(id0, it & 63u), p1 = __builtin_amdgcn_readlane(id1, it & 63u);
    const bool ok0 = p0 < a.n_pages, ok1 = p1 < a.n_pages;
    const bool whole = t0 + 32u <= s.hi && (t0 >= s.lo || t0 + 32u <= p.sinks);
    if (!(ok0 && ok1)) {  // an id that is not there hides its half; reported where an entry of it counts
      auto counts = [&](uint32_t t) { return t < s.hi && (t + 16u > s.lo || t < p.sinks); };
      if (lane == 0u && ((!ok0 && counts(t0)) || (!ok1 && counts(t0 + 16u)))) paged_flag(a.status);
      p0 = ok0 ? p0 : 0u;
      p1 = ok1 ? p1 : 0u;
    }
    Block<HD, F8> blk;
    blk.load(a, kv, col & 8u ? p1 : p0, g & 2u ? p1 : p0, t0, col, g);
    __builtin_amdgcn_sched_barrier(0);  // every load of the block before the first wait
    float sv[8];
    block_step<HD, F8>(blk, qb, c, t0 + 8u * g, s.hi, s.lo, s.hi, s.lo, p.sinks, g & 2u ? ok1 : ok0,
                       !(whole && ok0 && ok1), scale, sv, lane);
    if constexpr (WEIGHT) {
      if (col < p.G) {
        float4* to = reinterpret_cast<float4*>(p.scores + (static_cast<size_t>(b) * p.nh + kv * p.G + col) * p.vis + 32u * x + 8u * g);
        to[0] = make_float4(sv[0], sv[1], sv[2], sv[3]);
        to[1] = make_float4(sv[4], sv[5], sv[6], sv[7]);
      }
    }
  }
  c.l += lane_xor16_f32(c.l, lane);
  c.l += lane_xor32_f32(c.l, lane);
  if (lane < 16u) {
    s_ml[wave][col][0] = c.m;
    s_ml[wave][col][1] = c.l;
  }
#pragma unroll
  for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) s_o[wave][col][16u * nt + 4u * g + i] = c.o[nt][i];
  __syncthreads();
  for (uint32_t i = tid; i < p.G * HD; i += 256u) {
    const uint32_t h = i / HD, d = i % HD;
    float M = s_ml[0][h][0];
#pragma unroll
    for (uint32_t w = 1; w < 4; ++w) M = fmaxf(M, s_ml[w][h][0]);
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
      const float m = s_ml[w][h][0];
      const float fac = m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m - M);
      L = __builtin_fmaf(s_ml[w][h][1], fac, L);
      O = __builtin_fmaf(s_o[w][h][d], fac, O);
    }
    if (splits == 1u) {
      const float r = L == 0.0f ? 0.0f : O / L;
      p.out[(static_cast<size_t>(b) * p.nh + kv * p.G + h) * HD + d] = f32_to_bf16(F8 ? r * a.v_scale[kv] : r);
    } else {
      p.part[(static_cast<size_t>(blockIdx.x) * p.G + h) * HD + d] = O;
    }
    if (d == 0u && (splits > 1u || WEIGHT)) {
      p.ml[(static_cast<size_t>(blockIdx.x) * 16u + h) * 2u] = M;
      p.ml[(static_cast<size_t>(blockIdx.x) * 16u + h) * 2u + 1u] = L;
    }
  }
}

// The largest maximum of a head's parts and the sum taken to it, over a wave.
struct Total {
  float m, l;
};
__device__ __forceinline__ Total join_total(const float* ml, uint32_t splits, uint32_t lane) {
  float M = NEG_INF;
  for (uint32_t s = lane; s < splits; s += 64u) M = fmaxf(M, ml[s * 32u]);
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) M = fmaxf(M, __shfl_xor(M, k, 64));
  float L = 0.0f;
  for (uint32_t s = lane; s < splits; s += 64u) {
    const float m = ml[s * 32u];
    L = __builtin_fmaf(ml[s * 32u + 1u], m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m - M), L);
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) L += __shfl_xor(L, k, 64);
  return {M, L};
}

// Workgroups 0 .. n_seqs * nh - 1: a (sequence, head)'s parts joined in order.
// The others (WEIGHT): 1,024 listed entries of a (sequence, kv head) each, whose
// weights are the scores taken to the head's total.
template <uint32_t HD, bool F8, bool WEIGHT>
__global__ void __launch_bounds__(256) paged_join_kernel(Paged a, AttnArgs p, Weight w, uint32_t wchunks) {
  __shared__ float s_part[256 / HD][HD];
  __shared__ float s_tot[16][2];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const bool joins = blockIdx.x < a.n_seqs * p.nh;
  const uint32_t wi = blockIdx.x - a.n_seqs * p.nh;
  const uint32_t b = joins ? blockIdx.x / p.nh : wi / (a.n_kv * wchunks);
  const uint32_t kv = joins ? (blockIdx.x % p.nh) / p.G : wi / wchunks % a.n_kv;
  const uint32_t chunk = __builtin_amdgcn_readfirstlane(plan_chunk(a, p, lane));
  const Span s = decode_span(a, p, b);
  const uint32_t splits = plan_splits(s.nblk, chunk);
  if (joins) {
    if (splits == 1u) return;  // uniform: the part wrote the output
    const uint32_t h = blockIdx.x % p.nh, hh = h % p.G;
    const size_t first = plan_first(a, p, chunk, b, lane) + static_cast<size_t>(kv) * splits;
    const float* ml = p.ml + (first * 16u + hh) * 2u;
    const Total t = join_total(ml, splits, lane);
    const uint32_t d = tid % HD, part = tid / HD;
    float O = 0.0f;
    for (uint32_t i = part; i < splits; i += 256u / HD) {
      const float m = ml[i * 32u];
      O = __builtin_fmaf(p.part[((first + i) * p.G + hh) * HD + d], m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m - t.m), O);
    }
    s_part[part][d] = O;
    __syncthreads();
    if (tid < HD) {
      float sum = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < 256u / HD; ++i) sum += s_part[i][tid];
      const float r = t.l == 0.0f ? 0.0f : sum / t.l;
      p.out[(static_cast<size_t>(b) * p.nh + h) * HD + tid] = f32_to_bf16(F8 ? r * a.v_scale[kv] : r);
    }
    return;
  }
  if constexpr (WEIGHT) {
    const uint32_t c0 = 1024u * (wi % wchunks);
    if (c0 >= 32u * s.nblk) return;  // uniform
    const int64_t slot = weight_slot(w, b);
    if (slot < 0) {
      if (tid == 0u && kv == 0u && c0 == 0u) paged_flag(a.status);
      return;
    }
    const size_t first = plan_first(a, p, chunk, b, lane) + static_cast<size_t>(kv) * splits;
    for (uint32_t hh = wave; hh < p.G; hh += 4u) {
      const Total t = join_total(p.ml + (first * 16u + hh) * 2u, splits, lane);
      if (lane == 0u) {
        s_tot[hh][0] = t.m == NEG_INF ? 0.0f : t.m;
        s_tot[hh][1] = t.l == 0.0f ? 0.0f : 1.0f / t.l;
      }
    }
    __syncthreads();
    const uint32_t i0 = c0 + 4u * tid;
    if (i0 >= 32u * s.nblk) return;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t hh = 0; hh < p.G; ++hh) {
      const float4 sc = *reinterpret_cast<const float4*>(p.scores + (static_cast<size_t>(b) * p.nh + kv * p.G + hh) * p.vis + i0);
      const float m = s_tot[hh][0], r = s_tot[hh][1];
      sum[0] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc.x - m), r, sum[0]);
      sum[1] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc.y - m), r, sum[1]);
      sum[2] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc.z - m), r, sum[2]);
      sum[3] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc.w - m), r, sum[3]);
    }
    const uint32_t e0 = s.start(i0 / 32u) + i0 % 32u;
    float* to = w.w + (static_cast<size_t>(slot) * a.n_kv + kv) * w.ld;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t e = e0 + i;
      if (e < s.hi && (e >= s.lo || e < p.sinks)) to[e] += sum[i];
    }
  }
}

// ---------------------------------------------------------------------------
// Token rows of prompts
// ---------------------------------------------------------------------------
// A workgroup takes 256 / G consecutive rows of one sequence and the G heads of
// one kv head: 256 columns, 64 a wave (two groups of 32), over the blocks of 32
// entries that any of them sees (or a part of those, where there are few rows).
// Keys and values go through LDS, read there once per 64 columns: a block is
// 16 + 16 v_mfma_f32_32x32x16_bf16 (1,024 cycles of a SIMD) against 16 KB of LDS
// reads a wave (512 of the CU's cycles for the four).
//   S^T [32 entries x 32 columns] = K . Q^T, O^T [dims x 32 columns] += V^T . P: a
// lane (column lane % 32, half lane / 32) keeps its column throughout. Row r of
// the score tile is the block's entry with bits 2 and 3 of r exchanged, so a
// lane's sixteen scores are entries 8 half .. + 7 and 16 + 8 half .. + 7: the
// values of one 16-byte read of a transposed value row, in the order of the
// second product's operand.
// One wave has a SIMD to itself (512 registers), so products and softmax only
// overlap inside it: an iteration computes block x's softmax and value product
// together with block x + 1's scores, which do not depend on them. The running
// maximum follows the scores only when they pass it by 2^8 (the sums and O are
// in fp32 and P in bf16, which has fp32's range), so O is hardly ever rescaled.
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16_v;
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); }

constexpr uint32_t PF_COLS = 256, PF_TARGET = 512, PF_MIN_CHUNK = 8;
constexpr float PF_SLACK = 8.0f;

// Tiles and blocks of the sequences, as the parts are planned by.
struct PrefillSeq {
  uint32_t tiles, nblk;
};
__device__ __forceinline__ Span tile_span(const AttnArgs& p, const RowSpan& r, uint32_t n, uint32_t t0, uint32_t t1) {
  // entry of row t is n - (r1 - t); negative: nothing to see
  const uint32_t hi0 = n + t0 + 1u > r.r1 ? n + t0 + 1u - r.r1 : 0u, hi1 = n + t1 > r.r1 ? n + t1 - r.r1 : 0u;
  return span_of(hi0 ? hi0 - 1u : 0u, hi1, p.window, p.sinks);
}
__device__ __forceinline__ PrefillSeq prefill_seq(const Paged& a, const AttnArgs& p, uint32_t b) {
  const RowSpan r = paged_rows(a, b);
  const uint32_t tq = PF_COLS / p.G, tiles = (r.r1 - r.r0 + tq - 1u) / tq;
  return {tiles, tiles ? tile_span(p, r, paged_len(a, b), r.r0 + (tiles - 1u) * tq, r.r1).nblk : 0u};
}
struct PrefillItem {
  uint32_t b, tile, split, splits, chunk, first;  // first: the part of the tile's split 0
};
// Part `item` of a kv head: sequences in order, in each the last tile (the
// longest) first, a tile's parts together.
__device__ __forceinline__ PrefillItem prefill_find(const Paged& a, const AttnArgs& p, uint32_t item, uint32_t lane) {
  uint32_t chunk = 0xffffffffu;
  if (p.target) {  // few rows: parts of equal length
    uint64_t total = 0;
    for (uint32_t base = 0; base < a.n_seqs; base += 64u) {
      PrefillSeq s{0u, 0u};
      if (base + lane < a.n_seqs) s = prefill_seq(a, p, base + lane);
      total += wave_sum_u32(s.tiles * s.nblk);
    }
    chunk = uniform(max(PF_MIN_CHUNK, static_cast<uint32_t>((total * a.n_kv + p.target - 1u) / p.target)));
  }
  uint32_t acc = 0;
  for (uint32_t base = 0; base < a.n_seqs; base += 64u) {
    PrefillSeq s{0u, 0u};
    if (base + lane < a.n_seqs) s = prefill_seq(a, p, base + lane);
    const uint32_t splits = p.target ? plan_splits(s.nblk, chunk) : 1u;
    const uint32_t incl = wave_scan_u32(s.tiles * splits, lane), all = __builtin_amdgcn_readlane(incl, 63);
    if (item < acc + all) {
      const uint32_t l = static_cast<uint32_t>(__popcll(__ballot(acc + incl <= item)));
      const uint32_t before = acc + (l ? static_cast<uint32_t>(__builtin_amdgcn_readlane(incl, l - 1u)) : 0u);
      const uint32_t tl = __builtin_amdgcn_readlane(s.tiles, l), sp = __builtin_amdgcn_readlane(splits, l);
      const uint32_t x = (item - before) / sp, split = (item - before) % sp;
      return {uniform(base + l), uniform(tl - 1u - x), uniform(split), uniform(sp), uniform(chunk), uniform(item - split)};
    }
    acc += all;
  }
  return {a.n_seqs, 0u, 0u, 1u, chunk, 0u};
}

template <uint32_t HD, bool F8>
__global__ void __launch_bounds__(512) paged_prefill_kernel(Paged a, AttnArgs p) {
  constexpr uint32_t KS = HD / 16u, DT = HD / 32u, SZ = F8 ? 1u : 2u;
  constexpr uint32_t KROW = HD + 8u, VROW = 40u;  // padded rows (bf16): no bank is hit twice by eight lanes
  constexpr uint32_t KC = HD * SZ / 16u, VC = 2u * SZ;  // 16-byte chunks of a key row, of a block's value row
  constexpr uint32_t KN = 32u * KC, VN = HD * VC;       // chunks of a block: 512, 256 or 128, at most one a thread
  __shared__ __attribute__((aligned(16))) uint16_t s_k[2][32u * KROW];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[2][HD * VROW];
  __shared__ uint32_t s_bad;  // an edge block holds values that are not finite
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6);
  const uint32_t col = lane & 31u, half = lane >> 5;
  const uint32_t kv = blockIdx.x % a.n_kv;
  const PrefillItem it = prefill_find(a, p, blockIdx.x / a.n_kv, lane);
  const uint32_t b = it.b;
  if (b >= a.n_seqs) return;  // uniform
  // everything of the tile in scalar registers: no address or branch below takes the vector unit
  RowSpan r = paged_rows(a, b);
  r = {uniform(r.r0), uniform(r.r1)};
  const uint32_t n = uniform(paged_len(a, b));
  const uint32_t tq = PF_COLS / p.G, t0r = r.r0 + it.tile * tq, t1r = umin(r.r1, t0r + tq);
  if (tid == 0u && it.tile == 0u && it.split == 0u && kv == 0u && paged_len_bad(a, b)) paged_flag(a.status);
  const Span s = tile_span(p, r, n, t0r, t1r);
  const uint32_t hi_first = n + t0r + 1u > r.r1 ? n + t0r + 1u - r.r1 : 0u;
  const uint32_t lo_last = p.window && s.hi > p.window ? s.hi - p.window : 0u;
  const uint32_t x0 = it.split * (it.splits > 1u ? it.chunk : 0u);
  const uint32_t x1 = it.splits > 1u ? umin(s.nblk, x0 + it.chunk) : s.nblk;
  const float scale = F8 ? __uint_as_float(uniform(__float_as_uint(p.scale_log2 * a.k_scale[kv]))) : p.scale_log2;
  if (tid == 0u) s_bad = 0u;

  // the wave's columns: query slices, limits, state
  const uint32_t c = 32u * wave + col, t_row = t0r + c / p.G;
  const bool have = c / p.G < tq && t_row < t1r;
  const uint32_t hi = have && n + t_row + 1u > r.r1 ? n + t_row + 1u - r.r1 : 0u;
  const uint32_t lo = p.window && hi > p.window ? hi - p.window : 0u;
  bf16x8_v qb[KS];
  {
    const uint16_t* qr = p.q + static_cast<size_t>(have ? t_row : t0r) * p.q_ld + (kv * p.G + c % p.G) * HD + 8u * half;
#pragma unroll
    for (uint32_t ks = 0; ks < KS; ++ks) {
      u32x4_v v = *reinterpret_cast<const u32x4_v*>(qr + 16u * ks);
      if (!have) v = u32x4_v{0u, 0u, 0u, 0u};
      qb[ks] = __builtin_bit_cast(bf16x8_v, v);
    }
  }
  float m = NEG_INF, l = 0.0f;
  f32x16_v o[DT];
#pragma unroll
  for (uint32_t d = 0; d < DT; ++d) o[d] = f32x16_v{};

  // A wave's chunks lie in one half of a block, so in one page: a scalar offset
  // and a constant one a lane. Where a block has fewer chunks than threads, the
  // first waves bring keys and the last ones values.
  const uint32_t kc = tid, vc = VN == 512u ? tid : tid ^ 256u;
  const bool has_k = kc < KN, has_v = vc < VN;  // wave-uniform
  const uint32_t kh = uniform(kc / (KN / 2u)) & 1u, vh = uniform(vc / (VN / 2u)) & 1u;
  // A listed block: its first entry, whether its halves' page ids are good, the
  // (page, kv head) of the wave's keys and of its values, and whether any row
  // hides any of it. Behind the last block the last one again (unused).
  struct Blk {
    uint32_t t, ik, iv;
    bool ok0, ok1, edge;
  };
  const int32_t* table = a.table + static_cast<size_t>(b) * a.max_pages;
  const uint32_t pmask = (1u << a.lp) - 1u;
  uint32_t id0 = 0, id1 = 0;  // page ids of 64 blocks' halves, a block a lane
  auto fetch_ids = [&](uint32_t x) __attribute__((always_inline)) {
    const uint32_t t = s.start(umin(x + lane, s.nblk - 1u));
    id0 = static_cast<uint32_t>(table[umin(t >> a.lp, a.max_pages - 1u)]);
    id1 = static_cast<uint32_t>(table[umin((t + 16u) >> a.lp, a.max_pages - 1u)]);
  };
  auto block_of = [&](uint32_t x) __attribute__((always_inline)) {  // x within the 64 fetched last
    Blk k;
    k.t = s.start(umin(x, s.nblk - 1u));
    const uint32_t p0 = __builtin_amdgcn_readlane(id0, (x - x0) & 63u), p1 = __builtin_amdgcn_readlane(id1, (x - x0) & 63u);
    k.ok0 = p0 < a.n_pages;
    k.ok1 = p1 < a.n_pages;
    const uint32_t pk = kh ? p1 : p0, pv = vh ? p1 : p0;
    k.ik = (pk < a.n_pages ? pk : 0u) * a.n_kv + kv;
    k.iv = (pv < a.n_pages ? pv : 0u) * a.n_kv + kv;
    k.edge = !(k.ok0 && k.ok1 && k.t + 32u <= hi_first && (k.t >= lo_last || k.t + 32u <= p.sinks));
    return k;
  };
  const uint32_t v_dim = vc % (VN / 2u) / (VC / 2u), v_ent = 16u * vh + (16u / SZ) * (vc % (VC / 2u));
  const uint32_t koff = ((kc / KC) & pmask) * (HD * SZ) + 16u * (kc % KC);
  const uint32_t voff = ((v_dim << a.lp) + (v_ent & pmask)) * SZ;
  u32x4_v kr, vr;
  auto load_k = [&](const Blk& k) __attribute__((always_inline)) {
    const uint8_t* base = a.k + ((static_cast<size_t>(k.ik) << a.lp) + (k.t & pmask)) * (HD * SZ);
    if (KN == 512u || has_k) kr = *reinterpret_cast<const u32x4_v*>(base + koff);
  };
  auto load_v = [&](const Blk& k) __attribute__((always_inline)) {
    const uint8_t* base = a.v + ((static_cast<size_t>(k.iv) * HD << a.lp) + (k.t & pmask)) * SZ;
    if (VN == 512u || has_v) vr = *reinterpret_cast<const u32x4_v*>(base + voff);
  };
  // 16 stored bytes as bf16: one or two 16-byte words
  auto widen = [](const u32x4_v& w, uint32_t j) __attribute__((always_inline)) {
    if constexpr (F8) {
      const uint32_t w0 = j ? w.z : w.x, w1 = j ? w.w : w.y;
      return u32x4_v{e4m3x2_bf16<false>(w0), e4m3x2_bf16<true>(w0), e4m3x2_bf16<false>(w1), e4m3x2_bf16<true>(w1)};
    } else {
      return w;
    }
  };
  auto store_k = [&](uint32_t buf) __attribute__((always_inline)) {
    if (KN == 512u || has_k) {
      uint16_t* to = &s_k[buf][(kc / KC) * KROW + (16u / SZ) * (kc % KC)];
#pragma unroll
      for (uint32_t j = 0; j < 2u / SZ; ++j) *reinterpret_cast<u32x4_v*>(to + 8u * j) = widen(kr, j);
    }
  };
  // At the edge, values hidden from every row are stored as zero (the pool may
  // hold anything there), and those that are not finite too: the rows that see
  // them get them at the end, and no other row meets them.
  auto store_v = [&](uint32_t buf, const Blk& k) __attribute__((always_inline)) {
    if (VN == 512u || has_v) {
      u32x4_v w[2u / SZ];
#pragma unroll
      for (uint32_t j = 0; j < 2u / SZ; ++j) w[j] = widen(vr, j);
      if (k.edge) {  // uniform
        const bool ok = vh ? k.ok1 : k.ok0;
        bool bad = false;
#pragma unroll
        for (uint32_t j = 0; j < 2u / SZ; ++j) {
          w[j] &= entry_masks(k.t + v_ent + 8u * j, s.hi, s.lo, p.sinks, ok);
#pragma unroll
          for (uint32_t q = 0; q < 4; ++q) {
            const bool blo = (w[j][q] & 0x7f80u) == 0x7f80u, bhi = (w[j][q] & 0x7f800000u) == 0x7f800000u;
            bad = bad || blo || bhi;
            w[j][q] &= (blo ? 0u : 0xffffu) | (bhi ? 0u : 0xffff0000u);
          }
        }
        if (bad) s_bad = 1u;
      }
#pragma unroll
      for (uint32_t j = 0; j < 2u / SZ; ++j) *reinterpret_cast<u32x4_v*>(&s_v[buf][v_dim * VROW + v_ent + 8u * j]) = w[j];
    }
  };
  auto sees = [&](uint32_t e) __attribute__((always_inline)) { return e < hi && (e >= lo || e < p.sinks); };

  f32x16_v sa, sb;  // scores of this block and of the next, in turn
  float mx;
  const uint32_t krow = (col & 0x13u) | ((col & 4u) << 1) | ((col & 8u) >> 1);  // bits 2 and 3 exchanged
  auto scores = [&](uint32_t buf, f32x16_v& to) __attribute__((always_inline)) {
    to = f32x16_v{};
#pragma unroll
    for (uint32_t ks = 0; ks < KS; ++ks)
      to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          *reinterpret_cast<const bf16x8_v*>(&s_k[buf][krow * KROW + 16u * ks + 8u * half]), qb[ks], to, 0, 0, 0);
  };
  auto maximum = [&](const f32x16_v& v) __attribute__((always_inline)) {
    float t = fmaxf(v[0], v[1]);
#pragma unroll
    for (uint32_t i = 2; i < 16; i += 2) t = fmaxf(fmaxf(t, v[i]), v[i + 1]);
    mx = fmaxf(t, lane_xor32_f32(t, lane));
  };

  if (x0 < x1) {  // uniform
    fetch_ids(x0);
    Blk ka = block_of(x0), kb = block_of(x0 + 1u), kcb = block_of(x0 + 2u);
    load_k(ka);
    load_v(ka);
    __syncthreads();  // s_bad is zero
    store_k(x0 & 1u);
    store_v(x0 & 1u, ka);
    load_k(kb);
    store_k((x0 + 1u) & 1u);
    __syncthreads();
    scores(x0 & 1u, sa);
    maximum(sa);
    bool up = mx * scale > m + PF_SLACK;
    auto iteration = [&](uint32_t x, f32x16_v& sc, f32x16_v& next) __attribute__((always_inline)) {
      if (((x - x0) & 63u) == 61u) fetch_ids(x + 3u);  // uniform
      if (ka.edge) {  // uniform
        auto counts = [&](uint32_t e) { return e < s.hi && (e + 16u > s.lo || e < p.sinks); };
        if (tid == 0u && ((!ka.ok0 && counts(ka.t)) || (!ka.ok1 && counts(ka.t + 16u)))) paged_flag(a.status);
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i)
          sc[i] = (i < 8u ? ka.ok0 : ka.ok1) && sees(ka.t + 16u * (i / 8u) + 8u * half + i % 8u) ? sc[i] : NEG_INF;
        maximum(sc);
        up = mx * scale > m + PF_SLACK;
      }
      if (__any(up)) {
        const float mn = up ? mx * scale : m;
        const float f = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        m = mn;
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
          for (uint32_t i = 0; i < 16; ++i) o[d][i] *= f;
      }
      scores((x + 1u) & 1u, next);
      const float mu = m == NEG_INF ? 0.0f : m;
      typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
      const bf16x2_v ones = __builtin_bit_cast(bf16x2_v, 0x3f803f80u);
      bf16x8_v pb[2];
#pragma unroll
      for (uint32_t k2 = 0; k2 < 2; ++k2) {
        uint32_t pk[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          pk[i] = pack_bf16_pair_rne(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * k2 + 2 * i], scale, -mu)),
                                     __builtin_amdgcn_exp2f(__builtin_fmaf(sc[8 * k2 + 2 * i + 1], scale, -mu)));
          l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_v, pk[i]), ones, l, false);
        }
        pb[k2] = __builtin_bit_cast(bf16x8_v, u32x4_v{pk[0], pk[1], pk[2], pk[3]});
      }
      load_k(kcb);
      load_v(kb);
      __builtin_amdgcn_sched_barrier(0);  // the loads go out beside the scores' products, not behind the rest
#pragma unroll
      for (uint32_t k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              *reinterpret_cast<const bf16x8_v*>(&s_v[x & 1u][(32u * d + col) * VROW + 16u * k2 + 8u * half]), pb[k2], o[d], 0, 0, 0);
      maximum(next);
      up = mx * scale > m + PF_SLACK;
      const Blk kd = block_of(x + 3u);
      // K of x was read an iteration ago, V of x - 1 too: their buffers take K of x + 2 and V of x + 1
      store_k(x & 1u);
      store_v((x + 1u) & 1u, kb);
      __syncthreads();
      ka = kb;
      kb = kcb;
      kcb = kd;
    };
    for (uint32_t x = x0; x < x1; x += 2u) {
      iteration(x, sa, sb);
      if (x + 1u < x1) iteration(x + 1u, sb, sa);  // uniform
    }
    if (uniform(s_bad)) {  // after the last barrier; rare
      for (uint32_t x = x0; x < x1; ++x) {
        if (((x - x0) & 63u) == 0u) fetch_ids(x);
        const Blk k = block_of(x);
        if (!k.edge) continue;
        const uint32_t p0 = __builtin_amdgcn_readlane(id0, (x - x0) & 63u), p1 = __builtin_amdgcn_readlane(id1, (x - x0) & 63u);
        for (uint32_t i = 0; i < 32u; ++i) {
          const uint32_t e = k.t + i;
          if (!(i < 16u ? k.ok0 : k.ok1) || e >= s.hi) continue;
          const size_t base = (static_cast<size_t>(i < 16u ? p0 : p1) * a.n_kv + kv) * HD;
          const bool seen = sees(e);
#pragma unroll
          for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) {
              const size_t at = ((base + 32u * d + 8u * (j / 4u) + 4u * half + j % 4u) << a.lp) + (e & pmask);
              const uint32_t w = F8 ? e4m3x2_bf16<false>(a.v[at]) << 16
                                    : static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(a.v)[at]) << 16;
              const float v = (w & 0x7f800000u) == 0x7f800000u ? __uint_as_float(w) : 0.0f;
              o[d][j] += seen ? v : 0.0f;
            }
        }
      }
    }
  }
  const uint32_t h = kv * p.G + c % p.G;
  const float L = l + lane_xor32_f32(l, lane);
  if (!have) return;
  if (it.splits == 1u) {
    const float inv = (F8 ? a.v_scale[kv] : 1.0f) / L;
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
      for (uint32_t i = 0; i < 16; i += 4) {
        float v[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) v[j] = L == 0.0f ? 0.0f : o[d][i + j] * inv;
        *reinterpret_cast<uint2*>(p.out + (static_cast<size_t>(t_row) * p.nh + h) * HD + 32u * d + 2u * i + 4u * half) =
            make_uint2(pack_bf16_pair_rne(v[0], v[1]), pack_bf16_pair_rne(v[2], v[3]));
      }
  } else {
    const size_t at = static_cast<size_t>(blockIdx.x) * PF_COLS + c;
    if (half == 0u) {
      p.ml[at * 2u] = m;
      p.ml[at * 2u + 1u] = L;
    }
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d)
#pragma unroll
      for (uint32_t i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(p.part + at * HD + 32u * d + 2u * i + 4u * half) =
            make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
  }
}

// A tile's parts joined in order: a workgroup per 256 / HD * 4 columns.
template <uint32_t HD, bool F8>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(Paged a, AttnArgs p, uint32_t items) {
  constexpr uint32_t CW = 1024u / HD;  // columns of a workgroup, 4 dims a thread
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t part = blockIdx.x / (PF_COLS / CW), c = blockIdx.x % (PF_COLS / CW) * CW + tid / (HD / 4u), d = 4u * (tid % (HD / 4u));
  const uint32_t kv = part % a.n_kv;
  const PrefillItem it = prefill_find(a, p, part / a.n_kv, lane);
  if (it.b >= a.n_seqs || it.splits == 1u || it.split != 0u) return;  // uniform
  const RowSpan r = paged_rows(a, it.b);
  const uint32_t tq = PF_COLS / p.G, t = r.r0 + it.tile * tq + c / p.G, h = kv * p.G + c % p.G;
  if (c / p.G >= tq || t >= r.r1) return;
  float M = NEG_INF;
  for (uint32_t i = 0; i < it.splits; ++i)
    M = fmaxf(M, p.ml[((static_cast<size_t>(it.first + i) * a.n_kv + kv) * PF_COLS + c) * 2u]);
  float L = 0.0f;
  f32x4_v o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t i = 0; i < it.splits; ++i) {
    const size_t at = (static_cast<size_t>(it.first + i) * a.n_kv + kv) * PF_COLS + c;
    const float m = p.ml[at * 2u], f = m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m - M);
    const f32x4_v x = *reinterpret_cast<const f32x4_v*>(p.part + at * HD + d);
    L = __builtin_fmaf(p.ml[at * 2u + 1u], f, L);
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) o[j] = __builtin_fmaf(x[j], f, o[j]);
  }
  const float inv = (F8 ? a.v_scale[kv] : 1.0f) / L;
  float v[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) v[j] = L == 0.0f ? 0.0f : o[j] * inv;
  *reinterpret_cast<uint2*>(p.out + (static_cast<size_t>(t) * p.nh + h) * HD + d) =
      make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr uint32_t DECODE_TARGET = 1024, DECODE_MIN_CHUNK = 8;

// Blocks of 32 that a token can see of a sequence of `entries`.
uint64_t most_blocks(uint64_t entries, uint64_t window, uint32_t sinks) {
  const uint64_t all = (entries + 31u) / 32u;
  if (!window) return all;
  const uint64_t w = (window + 31u) / 32u + 1u + (std::min<uint64_t>(sinks, entries) + 31u) / 32u;
  return std::min(all, w);
}
struct DecodePlan {
  uint64_t items, vis, blocks;
  size_t ml, part, scores;  // bytes
};
size_t up256(size_t n) { return (n + 255u) & ~size_t(255); }
DecodePlan decode_plan(const obs_paged_kv* kv, const obs_paged_seqs* s, bool weight, uint32_t n_heads, uint32_t window,
                       uint32_t sinks) {
  DecodePlan d{};
  d.blocks = most_blocks(static_cast<uint64_t>(s->max_pages) * kv->page, window, sinks);
  d.vis = 32u * d.blocks;
  const uint64_t rows = static_cast<uint64_t>(s->n_seqs) * kv->n_kv;
  // sum of ceil(blocks / chunk) over the rows: at most target + rows, and at most each row's own most
  d.items = std::min<uint64_t>(DECODE_TARGET + rows, rows * ((d.blocks + DECODE_MIN_CHUNK - 1u) / DECODE_MIN_CHUNK));
  d.ml = up256(d.items * 32u * sizeof(float));
  d.part = up256(d.items * (n_heads / kv->n_kv) * kv->head_dim * sizeof(float));
  d.scores = weight ? up256(static_cast<size_t>(s->n_seqs) * n_heads * d.vis * sizeof(float)) : 0u;
  return d;
}

// Prefill: with few rows for the chip (tiles of both kinds of sequence ends
// counted by the rows alone) a tile's blocks are cut into parts.
struct PrefillPlan {
  uint64_t items;  // workgroups at most
  bool split;
  size_t ml, part;
};
PrefillPlan prefill_plan(const obs_paged_kv* kv, const obs_paged_seqs* s, uint32_t n_heads, uint32_t window, uint32_t sinks) {
  PrefillPlan d{};
  const uint32_t tq = PF_COLS / (n_heads / kv->n_kv);
  const uint64_t full = static_cast<uint64_t>(kv->n_kv) * ((s->n_rows + tq - 1u) / tq);
  // tiles: at most one that is not full a sequence, and none of a sequence without rows
  const uint64_t tiles = static_cast<uint64_t>(kv->n_kv) * std::min<uint64_t>(s->n_rows, (s->n_rows + tq - 1u) / tq + s->n_seqs);
  d.split = 2u * full <= PF_TARGET && most_blocks(static_cast<uint64_t>(s->max_pages) * kv->page, window ? static_cast<uint64_t>(window) + tq : 0u, sinks) > PF_MIN_CHUNK;
  d.items = d.split ? PF_TARGET + tiles : tiles;
  if (d.split) {
    d.ml = up256(d.items * PF_COLS * 2u * sizeof(float));
    d.part = up256(d.items * PF_COLS * kv->head_dim * sizeof(float));
  }
  return d;
}

int check_attn(obs_ctx* ctx, const char* who, const obs_paged_kv* kv, const obs_paged_seqs* seqs,
               const obs_kv_weight* weight, const uint16_t* q, const uint16_t* out, uint32_t n_heads, uint32_t* q_ld,
               const void* ws, size_t ws_bytes, size_t need) {
  if (!q || !out || !ws) return obs::set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
  if (weight) {
    const int rc = obs::check_weight(ctx, who, weight, static_cast<uint64_t>(seqs->max_pages) * kv->page, true);
    if (rc != OBS_OK) return rc;
  }
  *q_ld = *q_ld ? *q_ld : n_heads * kv->head_dim;
  if (*q_ld < n_heads * kv->head_dim || *q_ld % 8u)
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: q row stride %u must be a multiple of 8 holding a row", who, *q_ld);
  if (!obs::aligned(q, 16) || !obs::aligned(out, 16) || !obs::aligned(ws, 16))
    return obs::set_error(ctx, OBS_E_ALIGN, "%s: q, out and the workspace must be 16-byte aligned", who);
  if (ws_bytes < need) return obs::set_error(ctx, OBS_E_NOMEM, "%s: workspace %zu bytes < %zu needed", who, ws_bytes, need);
  return OBS_OK;
}

template <uint32_t HD, bool F8>
int launch_decode(obs_ctx* ctx, const Paged& a, const AttnArgs& p, const Weight& w, const DecodePlan& d) {
  const uint32_t grid = static_cast<uint32_t>(d.items), joins = a.n_seqs * p.nh;
  if (w.w) {
    OBS_LAUNCH(ctx, "paged_decode", paged_decode_kernel<HD, F8, true><<<grid, 256, 0, ctx->stream>>>(a, p));
    const uint32_t wchunks = static_cast<uint32_t>((d.vis + 1023u) / 1024u);
    OBS_LAUNCH(ctx, "paged_join", paged_join_kernel<HD, F8, true><<<joins + a.n_seqs * a.n_kv * wchunks, 256, 0, ctx->stream>>>(a, p, w, wchunks));
    return OBS_OK;
  }
  OBS_LAUNCH(ctx, "paged_decode", paged_decode_kernel<HD, F8, false><<<grid, 256, 0, ctx->stream>>>(a, p));
  if (d.blocks > DECODE_MIN_CHUNK)  // else every sequence is one part
    OBS_LAUNCH(ctx, "paged_join", paged_join_kernel<HD, F8, false><<<joins, 256, 0, ctx->stream>>>(a, p, w, 0u));
  return OBS_OK;
}

template <uint32_t HD, bool F8>
int launch_prefill(obs_ctx* ctx, const Paged& a, const AttnArgs& p, const PrefillPlan& d) {
  const uint32_t grid = static_cast<uint32_t>(d.items);
  OBS_LAUNCH(ctx, "paged_prefill", paged_prefill_kernel<HD, F8><<<grid, 512, 0, ctx->stream>>>(a, p));
  if (d.split)
    OBS_LAUNCH(ctx, "paged_prefill_join",
               paged_prefill_join_kernel<HD, F8><<<grid * (PF_COLS * HD / 1024u), 256, 0, ctx->stream>>>(a, p, grid));
  return OBS_OK;
}

}  // namespace

extern "C" {

int obs_sdpa_paged_workspace(obs_ctx* ctx, const obs_paged_kv* kv, const obs_paged_seqs* seqs,
                             const obs_kv_weight* weight, uint32_t n_heads, uint32_t window, uint32_t sinks,
                             size_t* bytes) {
  if (!ctx || !bytes) return OBS_E_INVALID;
  *bytes = 0;
  const char* who = "obs_sdpa_paged_workspace";
  int rc = obs::check_paged(ctx, who, kv, seqs, false);
  if (rc == OBS_OK) rc = obs::check_heads(ctx, who, n_heads, kv->n_kv);
  if (rc != OBS_OK) return rc;
  if (seqs->row) {
    const PrefillPlan f = prefill_plan(kv, seqs, n_heads, window, sinks);
    *bytes = f.ml + f.part + 256u;
  } else {
    const DecodePlan d = decode_plan(kv, seqs, weight != nullptr, n_heads, window, sinks);
    *bytes = d.ml + d.part + d.scores;
  }
  return OBS_OK;
}

int obs_sdpa_paged_decode(obs_ctx* ctx, const obs_paged_kv* kv, const obs_paged_seqs* seqs,
                          const obs_kv_weight* weight, const uint16_t* q, uint16_t* out, uint32_t n_heads,
                          uint32_t window, uint32_t sinks, uint32_t q_ld, void* ws, size_t ws_bytes) {
  if (!ctx) return OBS_E_INVALID;
  const char* who = "obs_sdpa_paged_decode";
  int rc = obs::check_paged(ctx, who, kv, seqs, true);
  if (rc == OBS_OK) rc = obs::check_heads(ctx, who, n_heads, kv->n_kv);
  if (rc != OBS_OK) return rc;
  if (seqs->row || seqs->n_rows != seqs->n_seqs)
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: one token a sequence (row NULL, n_rows == n_seqs); use obs_sdpa_paged_prefill", who);
  const DecodePlan d = decode_plan(kv, seqs, weight != nullptr, n_heads, window, sinks);
  rc = check_attn(ctx, who, kv, seqs, weight, q, out, n_heads, &q_ld, ws, ws_bytes, d.ml + d.part + d.scores);
  if (rc != OBS_OK) return rc;
  if (seqs->n_seqs == 0) return OBS_OK;
  const uint64_t grid = static_cast<uint64_t>(seqs->n_seqs) * (n_heads + kv->n_kv * ((d.vis + 1023u) / 1024u));
  if (d.items > 0x7fffffffull || grid > 0x7fffffffull)
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: too many sequences and heads", who);
  obs::DeviceGuard guard(ctx);
  const Paged a = obs::paged_args(ctx, kv, seqs);
  uint8_t* wb = static_cast<uint8_t*>(ws);
  const AttnArgs p{q, out, reinterpret_cast<float*>(wb), reinterpret_cast<float*>(wb + d.ml),
                   reinterpret_cast<float*>(wb + d.ml + d.part), n_heads, n_heads / kv->n_kv, window, sinks, q_ld,
                   static_cast<uint32_t>(d.vis), DECODE_MIN_CHUNK, DECODE_TARGET,
                   1.4426950408889634f / __builtin_sqrtf(static_cast<float>(kv->head_dim))};
  const Weight w = obs::weight_args(weight);
  const bool f8 = kv->dtype == OBS_KV_E4M3;
  if (kv->head_dim == 128u) return f8 ? launch_decode<128, true>(ctx, a, p, w, d) : launch_decode<128, false>(ctx, a, p, w, d);
  return f8 ? launch_decode<64, true>(ctx, a, p, w, d) : launch_decode<64, false>(ctx, a, p, w, d);
}

int obs_sdpa_paged_prefill(obs_ctx* ctx, const obs_paged_kv* kv, const obs_paged_seqs* seqs, const uint16_t* q,
                           uint16_t* out, uint32_t n_heads, uint32_t window, uint32_t sinks, uint32_t q_ld, void* ws,
                           size_t ws_bytes) {
  if (!ctx) return OBS_E_INVALID;
  const char* who = "obs_sdpa_paged_prefill";
  int rc = obs::check_paged(ctx, who, kv, seqs, true);
  if (rc == OBS_OK) rc = obs::check_heads(ctx, who, n_heads, kv->n_kv);
  if (rc != OBS_OK) return rc;
  if (!seqs->row) return obs::set_error(ctx, OBS_E_INVALID, "%s: null row (obs_sdpa_paged_decode takes one token a sequence)", who);
  const PrefillPlan d = prefill_plan(kv, seqs, n_heads, window, sinks);
  rc = check_attn(ctx, who, kv, seqs, nullptr, q, out, n_heads, &q_ld, ws, ws_bytes, d.ml + d.part + 256u);
  if (rc != OBS_OK) return rc;
  if (seqs->n_seqs == 0 || seqs->n_rows == 0) return OBS_OK;
  if (d.items * 32u > 0x7fffffffull) return obs::set_error(ctx, OBS_E_SHAPE, "%s: too many rows and heads", who);
  obs::DeviceGuard guard(ctx);
  const Paged a = obs::paged_args(ctx, kv, seqs);
  uint8_t* wb = static_cast<uint8_t*>(ws);
  const AttnArgs p{q, out, reinterpret_cast<float*>(wb), reinterpret_cast<float*>(wb + d.ml), nullptr, n_heads,
                   n_heads / kv->n_kv, window, sinks, q_ld, 0u, 0u, d.split ? PF_TARGET : 0u,
                   1.4426950408889634f / __builtin_sqrtf(static_cast<float>(kv->head_dim))};
  const bool f8 = kv->dtype == OBS_KV_E4M3;
  if (kv->head_dim == 128u) return f8 ? launch_prefill<128, true>(ctx, a, p, d) : launch_prefill<128, false>(ctx, a, p, d);
  return f8 ? launch_prefill<64, true>(ctx, a, p, d) : launch_prefill<64, false>(ctx, a, p, d);
}

}  // extern "C"
