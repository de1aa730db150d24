// obs_paged_attn.hip — attention of one new token of every sequence over a paged
// key/value cache (obs_sdpa_paged_decode), with a sliding window that keeps the
// first tokens visible, and the attention weight that entries gather.
#include "obs_paged.hpp"

namespace {
using namespace obsd;
using obs::Paged;
using obs::PagedAttn;
using obs::Weight;

// ---------------------------------------------------------------------------
// One block of 32 entries for one wave: 16 columns of queries
// ---------------------------------------------------------------------------
// S^T [32 entries x 16 columns] = K . Q^T by two v_mfma_f32_16x16x32_bf16 per 32
// dims, then O^T [dims x 16 columns] += V^T . P. A lane (col = lane % 16, g =
// lane / 16) ends with column col throughout, so every factor of the softmax is
// its own. Row r of score tile tt is entry 8 (r / 4) + 4 tt + r % 4 of the block:
// the lane's eight scores are then entries 8 g .. 8 g + 7, the eight values that
// one 16-byte load of a transposed value row brings.
// KEEP: values stay in the caches. From 64 entries on a row of a page holds several
// blocks' values in one line; below, they are streamed like the keys (32 sequences
// of up to 9,000, pages of 64: 69.5 us against 72.9 streamed, of 128 in e4m3 47.7
// and 54.4; of 32 48.2 and 43.7).
template <uint32_t HD, bool F8, bool KEEP>
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
      for (uint32_t i = 0; i < KL; ++i) k[tt][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_v*>(kr + 64u * i));
    }
    typedef typename std::conditional<F8, u32x2_v, u32x4_v>::type V;
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt) {
      const V* vr = reinterpret_cast<const V*>(vb + ((16u * nt + col) * SZ << a.lp));
      if constexpr (KEEP)
        v[nt] = *vr;
      else
        v[nt] = __builtin_nontemporal_load(vr);
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

// One block into the lane's column; t: the lane's first entry; hi, lo: what the
// token sees (values it does not see read as zero: the pool may hold anything
// there); ok: whether the lane's page is there; masked: whether the block needs
// any of it.
template <uint32_t HD, bool F8, bool KEEP>
__device__ __forceinline__ void block_step(const Block<HD, F8, KEEP>& blk, const bf16x8_v (&qb)[HD / 32u], Column<HD>& c,
                                           uint32_t t, uint32_t hi, uint32_t lo, uint32_t sinks, bool ok, bool masked,
                                           float scale_log2, float (&sv)[8], uint32_t lane) {
  constexpr uint32_t KS = HD / 32u, NT = HD / 16u;
#pragma unroll
  for (uint32_t tt = 0; tt < 2; ++tt) {
    f32x4_v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t ks = 0; ks < KS; ++ks) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(blk.key(tt, ks), qb[ks], acc, 0, 0, 0);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) sv[4 * tt + i] = acc[i] * scale_log2;
  }
  uint32_t bits = 0u;
  if (masked) {  // uniform
    bits = ok ? seen_bits(t, hi, lo, sinks) : 0u;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) sv[j] = bits >> j & 1u ? sv[j] : NEG_INF;
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
  if (masked) vm = word_masks(bits);
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
// Every sequence's blocks are cut into equal parts, so many that the call has
// about `target` (each of min_chunk blocks at least), by all lengths of the
// call: each wave adds them up itself, 64 sequences at a time.
__device__ __forceinline__ Span decode_span(const Paged& a, const PagedAttn& p, uint32_t b) {
  const uint32_t n = paged_len(a, b);
  return span_of(n ? n - 1u : 0u, n, p.window, p.sinks);
}
// Parts of a sequence: its share of the target, rounded up but for the rounding
// of the fp32 product, each of min_chunk blocks at least.
__device__ __forceinline__ uint32_t plan_parts(uint32_t nblk, float rate, uint32_t min_chunk) {
  const uint32_t share = static_cast<uint32_t>(__builtin_ceilf(static_cast<float>(nblk) * rate - 0.001f));
  return max(1u, umin(share, (nblk + min_chunk - 1u) / min_chunk));
}
// The sequence of part `item`, its entries, parts and first part; b is n_seqs
// behind the last. Up to 64 sequences the lengths are read once, a sequence a lane.
struct Found {
  uint32_t b, n, splits, first;
};
__device__ __forceinline__ uint32_t span_blocks(const PagedAttn& p, uint32_t n) {
  return span_of(n ? n - 1u : 0u, n, p.window, p.sinks).nblk;
}
// Parts a block. Where the target's parts would be short, those that the chip
// holds at once instead (DECODE_ONCE, less what rounding up adds): a second round
// costs more than it evens out (24 sequences of up to 4,000 26.7 -> 22.4 us, 64
// of 1,500 26.2 -> 22.8; but 48 of 6,000, 14 blocks a part, 52.0 against 56.4,
// and 256 of 2,000, 20 blocks, 94.9 against 103.8).
constexpr uint32_t DECODE_ONCE = 768;
__device__ __forceinline__ float plan_rate(const Paged& a, const PagedAttn& p, float total) {
  const float rows = static_cast<float>(a.n_seqs) * static_cast<float>(a.n_kv);
  const float work = fmaxf(total * static_cast<float>(a.n_kv), 1.0f);
  float target = static_cast<float>(p.target);
  if (p.target > DECODE_ONCE && work < (rows < 256.0f ? 9.5f : 16.0f) * target) target = fmaxf(DECODE_ONCE - 0.5f * rows, 128.0f);
  return target / work;
}
__device__ __forceinline__ Found plan_find(const Paged& a, const PagedAttn& p, uint32_t item, uint32_t lane) {
  float rate = 0.0f;
  uint32_t n = 0, nblk = 0;
  if (a.n_seqs <= 64u) {  // uniform
    n = lane < a.n_seqs ? paged_len(a, lane) : 0u;
    nblk = span_blocks(p, n);
    rate = plan_rate(a, p, static_cast<float>(wave_sum_u32(nblk)));
  } else {
    float total = 0.0f;
    for (uint32_t base = 0; base < a.n_seqs; base += 64u)
      total += static_cast<float>(wave_sum_u32(base + lane < a.n_seqs ? span_blocks(p, paged_len(a, base + lane)) : 0u));
    rate = plan_rate(a, p, total);
  }
  uint32_t acc = 0;
  for (uint32_t base = 0; base < a.n_seqs; base += 64u) {
    const uint32_t b = base + lane;
    if (a.n_seqs > 64u) {
      n = b < a.n_seqs ? paged_len(a, b) : 0u;
      nblk = span_blocks(p, n);
    }
    const uint32_t parts = plan_parts(nblk, rate, p.min_chunk);
    const uint32_t incl = wave_scan_u32(b < a.n_seqs ? a.n_kv * parts : 0u);
    const uint32_t all = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(incl), 63));
    if (item < acc + all) {
      const int l = static_cast<int>(__popcll(__ballot(acc + incl <= item)));
      const uint32_t end = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(incl), l));
      const uint32_t sp = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(parts), l));
      return {base + static_cast<uint32_t>(l), static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(n), l)), sp,
              acc + end - a.n_kv * sp};
    }
    acc += all;
  }
  return {a.n_seqs, 0u, 1u, 0u};
}

// ---------------------------------------------------------------------------
// One new token a sequence
// ---------------------------------------------------------------------------
// A workgroup takes one part of one (sequence, kv head); the G query heads are
// the columns. Its four waves take the part's blocks in turn and meet in LDS.
// A part that is all of its sequence writes the output, others their maximum,
// sum and output for paged_join_kernel.
template <uint32_t HD, bool F8, bool WEIGHT, bool KEEP>
__global__ void __launch_bounds__(256, 3) paged_decode_kernel(Paged a, PagedAttn p) {
  constexpr uint32_t NT = HD / 16u;
  __shared__ float s_ml[4][16][2];
  __shared__ float s_o[4][16][HD + 4u];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, col = lane & 15u, g = lane >> 4;
  const Found f = plan_find(a, p, blockIdx.x, lane);
  const uint32_t b = f.b, splits = f.splits, at = blockIdx.x - f.first;
  if (b >= a.n_seqs) return;  // uniform
  const Span s = span_of(f.n ? f.n - 1u : 0u, f.n, p.window, p.sinks);
  if (at == 0u && tid == 0u) p.plan[b] = make_uint2(blockIdx.x, splits);
  const uint32_t kv = at / splits, sp = at % splits;
  const uint32_t q0 = s.nblk / splits, q1 = s.nblk % splits;  // parts of q0 or q0 + 1 blocks
  const uint32_t x0 = sp * q0 + umin(sp, q1), x1 = x0 + q0 + (sp < q1 ? 1u : 0u);
  if (tid == 0u && at == 0u && paged_len_bad(a, b)) paged_flag(a.status);
  const float scale = F8 ? p.scale_log2 * a.k_scale[kv] : p.scale_log2;
  bf16x8_v qb[HD / 32u];
#pragma unroll
  for (uint32_t ks = 0; ks < HD / 32u; ++ks) {
    u32x4_v v = *reinterpret_cast<const u32x4_v*>(p.q + static_cast<size_t>(b) * p.q_ld + (kv * p.G + min(col, p.G - 1u)) * HD +
                                                  Block<HD, F8, KEEP>::q_dim(ks, g));
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
    Block<HD, F8, KEEP> blk;
    blk.load(a, kv, col & 8u ? p1 : p0, g & 2u ? p1 : p0, t0, col, g);
    __builtin_amdgcn_sched_barrier(0);  // every load of the block before the first wait
    float sv[8];
    block_step<HD, F8, KEEP>(blk, qb, c, t0 + 8u * g, s.hi, s.lo, p.sinks, g & 2u ? ok1 : ok0,
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
  M = wave_max_f32(M);
  float L = 0.0f;
  for (uint32_t s = lane; s < splits; s += 64u) {
    const float m = ml[s * 32u];
    L = __builtin_fmaf(ml[s * 32u + 1u], m == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m - M), L);
  }
  return {M, wave_sum_asc(L)};
}

// Workgroups 0 .. n_seqs * nh * HD / JD - 1: JD dims of a (sequence, head)'s
// parts joined in order (the plan, then maxima, sums and outputs of a round's
// parts in flight at once). The others (WEIGHT): 1,024 listed entries of a
// (sequence, kv head) each, whose weights are the scores taken to the head's
// total.
template <uint32_t HD, bool F8, bool WEIGHT, uint32_t JD>
__global__ void __launch_bounds__(256) paged_join_kernel(Paged a, PagedAttn p, Weight w, uint32_t wchunks) {
  constexpr uint32_t TD = JD / 4u, PT = 256u / TD, ROUND = 8u * PT;  // threads of a part, parts at once, parts a round
  __shared__ f32x4_v s_part[PT][TD];
  __shared__ float s_tot[16][2];
  __shared__ float s_fac[256];
  __shared__ float s_red[2][4];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  const uint32_t n_join = a.n_seqs * p.nh * (HD / JD);
  const bool joins = blockIdx.x < n_join;
  const uint32_t wi = blockIdx.x - n_join, head = blockIdx.x / (HD / JD);
  const uint32_t b = joins ? head / p.nh : wi / (a.n_kv * wchunks);
  const uint32_t kv = joins ? (head % p.nh) / p.G : wi / wchunks % a.n_kv;
  const uint2 plan = p.plan[b];
  const uint32_t splits = uniform(plan.y);
  const size_t first = static_cast<size_t>(uniform(plan.x)) + static_cast<size_t>(kv) * splits;
  if (joins) {
    if (splits == 1u) return;  // uniform: the part wrote the output
    const uint32_t h = head % p.nh, hh = h % p.G, d = tid % TD, row = tid / TD, d0 = JD * (blockIdx.x % (HD / JD));
    const float* ml = p.ml + (first * 16u + hh) * 2u;
    const float* part = p.part + (first * p.G + hh) * HD + d0 + 4u * d;
    float M = NEG_INF, L = 0.0f;
    f32x4_v acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t s0 = 0; s0 < splits; s0 += ROUND) {
      const uint32_t cnt = umin(ROUND, splits - s0);
      const float2 own = tid < cnt ? *reinterpret_cast<const float2*>(ml + (s0 + tid) * 32u) : make_float2(NEG_INF, 0.0f);
      f32x4_v x[8];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        x[i] = row + PT * i < cnt ? *reinterpret_cast<const f32x4_v*>(part + static_cast<size_t>(s0 + row + PT * i) * p.G * HD)
                                  : f32x4_v{0.0f, 0.0f, 0.0f, 0.0f};
      const float wm = wave_max_f32(own.x);
      if (s0) __syncthreads();  // what the round before left in LDS was read
      if (lane == 0u) s_red[0][wave] = wm;
      __syncthreads();
      const float mn = fmaxf(fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3])), M);
      const float back = M == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(M - mn);
      const float fac = own.x == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(own.x - mn);
      const float wl = wave_sum_asc(own.y * fac);
      s_fac[tid] = fac;
      if (lane == 0u) s_red[1][wave] = wl;
      __syncthreads();
      M = mn;
      L = __builtin_fmaf(L, back, (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]));
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) acc[j] *= back;
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const float f = s_fac[row + PT * i];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(x[i][j], f, acc[j]);
      }
    }
    s_part[row][d] = acc;
    __syncthreads();
    if (tid < JD) {
      const float* col = reinterpret_cast<const float*>(&s_part[0][0]) + tid;
      float sum = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < PT; ++i) sum += col[JD * i];
      const float r = L == 0.0f ? 0.0f : sum * ((F8 ? a.v_scale[kv] : 1.0f) / L);
      p.out[(static_cast<size_t>(b) * p.nh + h) * HD + d0 + tid] = f32_to_bf16(r);
    }
    return;
  }
  if constexpr (WEIGHT) {
    const Span s = decode_span(a, p, b);
    const uint32_t c0 = 1024u * (wi % wchunks);
    if (c0 >= 32u * s.nblk) return;  // uniform
    const int64_t slot = weight_slot(w, b);
    if (slot < 0) {
      if (tid == 0u && kv == 0u && c0 == 0u) paged_flag(a.status);
      return;
    }
    // the first heads' scores and the entries' weights are requested before the totals
    const uint32_t i0 = c0 + 4u * tid, ic = umin(i0, 32u * s.nblk - 4u), e0 = s.start(ic / 32u) + ic % 32u;
    const float* sc0 = p.scores + (static_cast<size_t>(b) * p.nh + kv * p.G) * p.vis + ic;
    float* to = w.w + (static_cast<size_t>(slot) * a.n_kv + kv) * w.ld;
    auto sees = [&](uint32_t e) { return i0 < 32u * s.nblk && e < s.hi && (e >= s.lo || e < p.sinks); };
    float4 sc[8];
    float old[4];
    auto scores_from = [&](uint32_t h0) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) sc[i] = *reinterpret_cast<const float4*>(sc0 + static_cast<size_t>(umin(h0 + i, p.G - 1u)) * p.vis);
    };
    scores_from(0u);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) old[i] = sees(e0 + i) ? to[e0 + i] : 0.0f;
    for (uint32_t hh = wave; hh < p.G; hh += 4u) {
      const Total t = join_total(p.ml + (first * 16u + hh) * 2u, splits, lane);
      if (lane == 0u) {
        s_tot[hh][0] = t.m == NEG_INF ? 0.0f : t.m;
        s_tot[hh][1] = t.l == 0.0f ? 0.0f : 1.0f / t.l;
      }
    }
    __syncthreads();
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t h0 = 0; h0 < p.G; h0 += 8u) {
      if (h0) scores_from(h0);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const float m = s_tot[umin(h0 + i, p.G - 1u)][0], r = h0 + i < p.G ? s_tot[h0 + i][1] : 0.0f;
        sum[0] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc[i].x - m), r, sum[0]);
        sum[1] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc[i].y - m), r, sum[1]);
        sum[2] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc[i].z - m), r, sum[2]);
        sum[3] = __builtin_fmaf(__builtin_amdgcn_exp2f(sc[i].w - m), r, sum[3]);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
      if (sees(e0 + i)) to[e0 + i] = old[i] + sum[i];
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr uint32_t DECODE_MIN_CHUNK = 4;
// Blocks up to which a sequence is one part where no weight is gathered (no join
// then), by what the page table can hold, as the lengths are the device's: a table of
// 32,768 entries takes one sequence of 256 from 6.6 to 9.0 us, 64 of 1,000 from 24.2 to
// 30.4 and, with weights, 16 of up to 8,200 from 34.4 to 40.8 (the join's workgroups
// are as many as the table has entries for). In tables as long as the sequences, parts and their join cost more up to 384 entries (one sequence of 256
// 8.9 us in parts, 6.8 whole; of 384 8.9 and 8.2, of 512 8.9 and 9.4), more rows
// fill the chip by themselves (48 of 512 12.8 and 11.7; 64 of 1,000 22.3 and
// 19.7, of 2,000 32.3 and 34.6; 32 of 1,000 12.8 and 18.4), and blocks in e4m3
// are half as long (256 of 2,000 59.8 and 56.1, in bf16 94.9 and 99.3).
uint32_t decode_whole(uint64_t rows, bool f8) { return rows >= 512u && f8 ? 64u : rows >= 256u ? 32u : rows >= 96u ? 16u : 12u; }
// Parts of a call: three workgroups a CU are resident (DECODE_ONCE). Few rows give
// nearly equal parts, which fill the chip once (one sequence of 100,003 entries
// 46.6 us against 52.8 with 1,152); the parts of many sequences differ, and
// finer ones even out (48 sequences of up to 16,000: 72.3 us against 74.6).
uint32_t decode_target(const obs_paged_kv* kv, const obs_paged_seqs* s) { return s->n_seqs * kv->n_kv <= 32u ? DECODE_ONCE : 1152u; }

struct DecodePlan {
  uint64_t items, vis, blocks;
  size_t ml, part, scores, plan;  // bytes
  uint32_t min_chunk;
  size_t all() const { return ml + part + scores + plan; }
};
using obs::most_blocks;
using obs::up256;

DecodePlan decode_plan(const obs_paged_kv* kv, const obs_paged_seqs* s, bool weight, uint32_t n_heads, uint32_t window,
                       uint32_t sinks) {
  DecodePlan d{};
  d.blocks = most_blocks(static_cast<uint64_t>(s->max_pages) * kv->page, window, sinks);
  d.vis = 32u * d.blocks;
  const uint64_t rows = static_cast<uint64_t>(s->n_seqs) * kv->n_kv;
  const uint32_t whole = weight ? 0u : decode_whole(rows, kv->dtype == OBS_KV_E4M3);
  d.min_chunk = std::max(DECODE_MIN_CHUNK, d.blocks <= whole ? whole : 0u);
  // sum of the rows' rounded shares: at most target + rows (and what fp32 rounds), and at most each row's own most
  d.items = std::min<uint64_t>(decode_target(kv, s) + rows + 64u, rows * ((d.blocks + d.min_chunk - 1u) / d.min_chunk));
  d.ml = up256(d.items * 32u * sizeof(float));
  d.part = up256(d.items * (n_heads / kv->n_kv) * kv->head_dim * sizeof(float));
  d.scores = weight ? up256(static_cast<size_t>(s->n_seqs) * n_heads * d.vis * sizeof(float)) : 0u;
  d.plan = up256(s->n_seqs * sizeof(uint2));
  return d;
}

template <uint32_t HD, bool F8, bool WEIGHT>
int launch_decode(obs_ctx* ctx, const Paged& a, const PagedAttn& p, const Weight& w, const DecodePlan& d) {
  const uint32_t items = static_cast<uint32_t>(d.items);
  if (a.lp >= 6u)
    OBS_LAUNCH(ctx, "paged_decode", paged_decode_kernel<HD, F8, WEIGHT, true><<<items, 256, 0, ctx->stream>>>(a, p));
  else
    OBS_LAUNCH(ctx, "paged_decode", paged_decode_kernel<HD, F8, WEIGHT, false><<<items, 256, 0, ctx->stream>>>(a, p));
  if (!WEIGHT && d.blocks <= d.min_chunk) return OBS_OK;  // every sequence is one part
  const uint32_t wchunks = WEIGHT ? static_cast<uint32_t>((d.vis + 1023u) / 1024u) : 0u, rows = a.n_seqs * p.nh;
  const uint32_t weights = rows / p.G * wchunks;
  // few rows have many parts each: four workgroups a row (one sequence of 100,003
  // entries 46.5 us against 48.2; 48 sequences of up to 16,000 77.7 against 72.3)
  if (rows < 256u)
    OBS_LAUNCH(ctx, "paged_join",
               paged_join_kernel<HD, F8, WEIGHT, 32><<<rows * (HD / 32u) + weights, 256, 0, ctx->stream>>>(a, p, w, wchunks));
  else
    OBS_LAUNCH(ctx, "paged_join", paged_join_kernel<HD, F8, WEIGHT, HD><<<rows + weights, 256, 0, ctx->stream>>>(a, p, w, wchunks));
  return OBS_OK;
}

}  // namespace

namespace obs {
int check_attn(obs_ctx* ctx, const char* who, const obs_paged_kv* kv, const obs_paged_seqs* seqs,
               const obs_kv_weight* weight, const uint16_t* q, const uint16_t* out, uint32_t n_heads, uint32_t* q_ld,
               const void* ws, size_t ws_bytes, size_t need) {
  if (!q || !out || (!ws && need)) return set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
  if (weight) {
    const int rc = check_weight(ctx, who, weight, static_cast<uint64_t>(seqs->max_pages) * kv->page, true);
    if (rc != OBS_OK) return rc;
  }
  *q_ld = *q_ld ? *q_ld : n_heads * kv->head_dim;
  if (*q_ld < n_heads * kv->head_dim || *q_ld % 8u)
    return set_error(ctx, OBS_E_SHAPE, "%s: q row stride %u must be a multiple of 8 holding a row", who, *q_ld);
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(ws, 16))
    return set_error(ctx, OBS_E_ALIGN, "%s: q, out and the workspace must be 16-byte aligned", who);
  if (ws_bytes < need) return set_error(ctx, OBS_E_NOMEM, "%s: workspace %zu bytes < %zu needed", who, ws_bytes, need);
  return OBS_OK;
}

}  // namespace obs

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
    *bytes = obs::prefill_paged_ws(kv, seqs, n_heads, window, sinks);
  } else {
    const DecodePlan d = decode_plan(kv, seqs, weight != nullptr, n_heads, window, sinks);
    *bytes = d.all();
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
  rc = obs::check_attn(ctx, who, kv, seqs, weight, q, out, n_heads, &q_ld, ws, ws_bytes, d.all());
  if (rc != OBS_OK) return rc;
  if (seqs->n_seqs == 0) return OBS_OK;
  const uint64_t wchunks = weight ? (d.vis + 1023u) / 1024u : 0u;
  rc = obs::check_grid(ctx, who, std::max(d.items, seqs->n_seqs * (static_cast<uint64_t>(n_heads) * 4u + kv->n_kv * wchunks)), 256u);
  if (rc != OBS_OK) return rc;
  obs::DeviceGuard guard(ctx);
  const Paged a = obs::paged_args(ctx, kv, seqs);
  uint8_t* wb = static_cast<uint8_t*>(ws);
  const PagedAttn p{q, out, reinterpret_cast<float*>(wb), reinterpret_cast<float*>(wb + d.ml),
                   reinterpret_cast<float*>(wb + d.ml + d.part), reinterpret_cast<uint2*>(wb + d.ml + d.part + d.scores),
                   n_heads, n_heads / kv->n_kv, window, sinks, q_ld,
                   static_cast<uint32_t>(d.vis), d.min_chunk, decode_target(kv, seqs), 0u,
                   1.4426950408889634f / __builtin_sqrtf(static_cast<float>(kv->head_dim))};
  const Weight w = obs::weight_args(weight);
  const bool f8 = kv->dtype == OBS_KV_E4M3;
  if (kv->head_dim == 128u) {
    if (weight) return f8 ? launch_decode<128, true, true>(ctx, a, p, w, d) : launch_decode<128, false, true>(ctx, a, p, w, d);
    return f8 ? launch_decode<128, true, false>(ctx, a, p, w, d) : launch_decode<128, false, false>(ctx, a, p, w, d);
  }
  if (weight) return f8 ? launch_decode<64, true, true>(ctx, a, p, w, d) : launch_decode<64, false, true>(ctx, a, p, w, d);
  return f8 ? launch_decode<64, true, false>(ctx, a, p, w, d) : launch_decode<64, false, false>(ctx, a, p, w, d);
}

}  // extern "C"
