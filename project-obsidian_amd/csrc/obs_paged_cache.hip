// obs_paged_cache.hip — a paged key/value cache of several sequences: the
// checks of its arguments, q/k norm + RoPE + append (obs_attn_prep_paged) and
// the eviction by gathered attention weight (obs_kv_evict).
#include "obs_paged.hpp"

namespace {
using namespace obsd;
using obs::Paged;
using obs::Weight;

// ---------------------------------------------------------------------------
// q/k RMSNorm + NeoX RoPE + append
// ---------------------------------------------------------------------------
// The sequence that token row t belongs to: the number of ends row[1..n_seqs]
// at or below t, counted by a wave (64 ends at once, or 64 ends of 64 each and
// then one such block). n_seqs and above: behind the last sequence.
__device__ __forceinline__ uint32_t seq_of_row(const Paged& a, uint32_t t, uint32_t lane) {
  if (!a.row) return t;
  uint32_t base = 0u;
  if (a.n_seqs > 64u) {
    const uint32_t blocks = (a.n_seqs + 63u) / 64u;  // <= 64
    const int32_t end = a.row[min(64u * (min(lane, blocks - 1u) + 1u), a.n_seqs)];
    base = 64u * static_cast<uint32_t>(__popcll(__ballot(lane < blocks && end <= static_cast<int32_t>(t))));
    if (base >= a.n_seqs) return a.n_seqs;
  }
  const uint32_t b = base + lane;
  const int32_t end = a.row[min(b, a.n_seqs - 1u) + 1u];
  return base + static_cast<uint32_t>(__popcll(__ballot(b < a.n_seqs && end <= static_cast<int32_t>(t))));
}

struct PrepArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  uint16_t* q_out;
  const int32_t* pos;
  const float* rope;
  uint32_t nh, rope_len, q_ld, kv_ld, q_out_ld;
  float eps;
};

// The sequence of row t for a lane of its own: a search over the ends from
// sequence lo on (the first one that ends behind t).
__device__ __forceinline__ uint32_t seq_of_row_lane(const Paged& a, uint32_t t, uint32_t lo) {
  uint32_t hi = a.n_seqs;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2u;
    if (a.row[mid + 1u] <= static_cast<int32_t>(t))
      lo = mid + 1u;
    else
      hi = mid;
  }
  return lo;
}

// Values of 64 consecutive token rows of one kv head, transposed through LDS:
// a lane owns a row, so a store of one dim writes the runs of consecutive
// entries that the rows are. (From each row's own workgroup, one entry of a
// cache row at a time, the stores cost more than everything else: 38.8 against
// 28.3 us for 5,795 rows into an e4m3 cache.)
constexpr uint32_t PREP_TILE = 64;
template <uint32_t HD, bool F8>
__device__ __forceinline__ void prep_paged_values(const Paged& a, const PrepArgs& p, uint32_t vi) {
  __shared__ uint32_t s_v[PREP_TILE][HD / 2u + 1u];  // rows of dim pairs (+1 word: bank spread)
  const uint32_t h = vi % a.n_kv, t0 = vi / a.n_kv * PREP_TILE, nt = umin(PREP_TILE, a.n_rows - t0);
#pragma unroll
  for (uint32_t i = 0; i < PREP_TILE * HD / 2048u; ++i) {  // 16-byte chunks
    const uint32_t c = threadIdx.x + 256u * i, r = c / (HD / 8u), d = 8u * (c % (HD / 8u));
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (r < nt) x = *reinterpret_cast<const uint4*>(p.v + static_cast<size_t>(t0 + r) * p.kv_ld + h * HD + d);
    uint32_t* to = &s_v[r][d / 2u];
    to[0] = x.x;
    to[1] = x.y;
    to[2] = x.z;
    to[3] = x.w;
  }
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, t = t0 + lane;
  const uint32_t b0 = seq_of_row(a, t0, lane);
  bool there = false;
  size_t at = 0;
  if (lane < nt && b0 < a.n_seqs) {
    const uint32_t b = seq_of_row_lane(a, t, b0);
    if (b < a.n_seqs) {
      const RowSpan r = paged_rows(a, b);
      const int32_t entry = static_cast<int32_t>(paged_len(a, b)) - static_cast<int32_t>(r.r1 - t);
      const int32_t pos = p.pos ? p.pos[t] : entry;
      if (t >= r.r0 && t < r.r1 && entry >= 0 && pos >= 0 && static_cast<uint32_t>(pos) < p.rope_len) {
        const uint32_t page = paged_id(a, b, static_cast<uint32_t>(entry), there);  // reported by the row's workgroup
        at = ((static_cast<size_t>(page) * a.n_kv + h) * HD << a.lp) + (static_cast<uint32_t>(entry) & ((1u << a.lp) - 1u));
      }
    }
  }
  const float s = F8 ? a.v_scale[h] : 1.0f;
  __syncthreads();
  if (!there) return;
  for (uint32_t d = wave * (HD / 4u); d < (wave + 1u) * (HD / 4u); d += 2u) {
    const uint32_t w = s_v[lane][d / 2u];
    if constexpr (F8) {
      const uint32_t b2 = pack_e4m3x4(bf16lo(w) / s, bf16hi(w) / s, 0.0f, 0.0f);
      uint8_t* to = const_cast<uint8_t*>(a.v) + at + (static_cast<size_t>(d) << a.lp);
      to[0] = static_cast<uint8_t>(b2);
      to[1u << a.lp] = static_cast<uint8_t>(b2 >> 8);
    } else {
      uint16_t* to = reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(a.v)) + at + (static_cast<size_t>(d) << a.lp);
      to[0] = static_cast<uint16_t>(w);
      to[1u << a.lp] = static_cast<uint16_t>(w >> 16);
    }
  }
}

// Workgroups 0 .. n_vt - 1 bring the values of prompts (none with one token a
// sequence). The others: one token row each, or four; HD / 8 lanes per head with 8 dims
// each, so a wave norms and rotates 512 / HD heads at once. The sums and the
// rotation are attn_prep_rows_kernel's, in its order. The first heads are
// requested before the row's sequence, entry and position are known.
template <uint32_t HD, bool F8, uint32_t WAVES>
__global__ void __launch_bounds__(256, 8) prep_paged_kernel(Paged a, PrepArgs p, Weight w, uint32_t n_vt) {
  constexpr uint32_t LPH = HD / 8u, HPW = 64u / LPH;  // lanes per head, heads per wave
  if (blockIdx.x < n_vt) {  // uniform
    prep_paged_values<HD, F8>(a, p, blockIdx.x);
    return;
  }
  const uint32_t lane = threadIdx.x & 63u, m = lane % LPH, c0 = 8u * m;
  const uint32_t w4 = uniform(threadIdx.x >> 6), wave = w4 % WAVES;           // the wave among its row's
  const uint32_t tid = threadIdx.x % (64u * WAVES), threads = 64u * WAVES;  // the thread among its row's
  const uint32_t t = (blockIdx.x - n_vt) * (4u / WAVES) + w4 / WAVES, heads = p.nh + a.n_kv;
  if (t >= a.n_rows) return;  // uniform per wave, as all below (no barrier)
  const uint16_t* q = p.q + static_cast<size_t>(t) * p.q_ld;
  const uint16_t* k = p.k + static_cast<size_t>(t) * p.kv_ld;
  auto load_head = [&](uint32_t head) __attribute__((always_inline)) {  // clamped: past the last head, unused
    const uint32_t hc = umin(head, heads - 1u);
    return *reinterpret_cast<const uint4*>((hc < p.nh ? q + hc * HD : k + (hc - p.nh) * HD) + c0);
  };
  uint4 xv = load_head(HPW * wave + lane / LPH);
  const uint4 wq = *reinterpret_cast<const uint4*>(p.q_norm + c0), wk = *reinterpret_cast<const uint4*>(p.k_norm + c0);
  const uint32_t b = uniform(seq_of_row(a, t, lane));
  if (b >= a.n_seqs) return;  // uniform
  const RowSpan rs = paged_rows(a, b);
  if (t < rs.r0 || t >= rs.r1) return;
  const uint32_t n = uniform(paged_len(a, b));
  if (t == rs.r0 && tid == 0u && paged_len_bad(a, b)) paged_flag(a.status);
  const int32_t entry = static_cast<int32_t>(n) - static_cast<int32_t>(uniform(rs.r1) - t);
  const int32_t pos = p.pos ? static_cast<int32_t>(uniform(static_cast<uint32_t>(p.pos[t]))) : entry;
  if (pos < 0 || static_cast<uint32_t>(pos) >= p.rope_len) {  // uniform
    // without positions of the caller's own it is the length that is out of range
    if (!p.pos && entry >= 0 && tid == 0u) paged_flag(a.status);
    return;
  }
  float cs[8], sn[8];  // of the lane's pairs: columns c0 .. c0 + 7 modulo HD / 2
  {
    const float* tab = p.rope + static_cast<size_t>(pos) * 128u + (HD == 128u ? 16u : 32u) * (m % (LPH / 2u));
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      // the table's pair i has theta^(-2i/128); a head of 64 takes every second one
      const float2 t2 = *reinterpret_cast<const float2*>(tab + (HD == 128u ? 2u : 4u) * i);
      cs[i] = t2.x;
      sn[i] = t2.y;
    }
  }
  bool there = entry >= 0;
  const uint32_t e = there ? static_cast<uint32_t>(entry) : 0u;
  bool ok;
  const uint32_t page = uniform(paged_id(a, b, e, ok));
  if (there && !ok && tid == 0u) paged_flag(a.status);
  there = there && ok;
  const uint32_t off = e & ((1u << a.lp) - 1u);
  if (w.w && entry >= 0 && tid < a.n_kv) {
    const int64_t s = weight_slot(w, b);
    if (s >= 0)
      for (uint32_t h = tid; h < a.n_kv; h += threads) w.w[(static_cast<size_t>(s) * a.n_kv + h) * w.ld + e] = 0.0f;
    else if (tid == 0u)
      paged_flag(a.status);
  }
  uint16_t* q_out = p.q_out + static_cast<size_t>(t) * p.q_out_ld;
  const size_t page0 = static_cast<size_t>(page) * a.n_kv;
  const uint32_t pg = 1u << a.lp;
  const bool first = m < LPH / 2u;
  for (uint32_t hb = HPW * wave; hb < heads; hb += WAVES * HPW) {  // uniform per wave
    const uint32_t head = hb + lane / LPH;
    const bool is_q = head < p.nh;
    const uint4 xnext = load_head(head + WAVES * HPW);
    const uint32_t xw[4] = {xv.x, xv.y, xv.z, xv.w};
    const uint32_t ww[4] = {is_q ? wq.x : wk.x, is_q ? wq.y : wk.y, is_q ? wq.z : wk.z, is_q ? wq.w : wk.w};
    xv = xnext;
    float ps[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const float x0 = bf16lo(xw[i]), x1 = bf16hi(xw[i]);
      ps[i] = __builtin_fmaf(x0, x0, 0.0f);
      ps[i] = __builtin_fmaf(x1, x1, ps[i]);
    }
    float ss = (ps[0] + ps[1]) + (ps[2] + ps[3]);
    ss = ss + dpp_f32<DPP_XOR1>(ss);
    ss = ss + dpp_f32<DPP_XOR2>(ss);
    ss = ss + dpp_f32<DPP_HALF_MIRROR>(ss);
    if constexpr (HD == 128u) ss = ss + dpp_f32<DPP_MIRROR>(ss);
    const float inv = 1.0f / __builtin_sqrtf(ss / static_cast<float>(HD) + p.eps);
    float nvs[8], r[8];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const float n0 = (bf16lo(xw[i]) * inv) * bf16lo(ww[i]), n1 = (bf16hi(xw[i]) * inv) * bf16hi(ww[i]);
      // what becomes bf16 is rounded as the stored q / k would be; a key in e4m3 only at its end
      const uint32_t pr = pack_bf16_pair_rne(n0, n1);
      nvs[2 * i] = F8 && !is_q ? n0 : bf16lo(pr);
      nvs[2 * i + 1] = F8 && !is_q ? n1 : bf16hi(pr);
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const float nv = nvs[i];
      float other;  // columns +- HD / 2
      if constexpr (HD == 128u)
        other = dpp_f32<DPP_ROW_ROR8>(nv);
      else
        other = dpp_xor4_f32(nv);
      const float x0 = nv * cs[i], x1 = other * sn[i];
      r[i] = first ? x0 - x1 : x0 + x1;
    }
    if (head >= heads) continue;
    if (is_q) {
      *reinterpret_cast<uint4*>(q_out + head * HD + c0) =
          make_uint4(pack_bf16_pair_rne(r[0], r[1]), pack_bf16_pair_rne(r[2], r[3]), pack_bf16_pair_rne(r[4], r[5]),
                     pack_bf16_pair_rne(r[6], r[7]));
    } else if (there) {
      const uint32_t h = head - p.nh;
      const size_t at = ((page0 + h) * pg + off) * HD + c0;
      if constexpr (F8) {
        const float s = a.k_scale[h];
        uint2 o;
        o.x = pack_e4m3x4(r[0] / s, r[1] / s, r[2] / s, r[3] / s);
        o.y = pack_e4m3x4(r[4] / s, r[5] / s, r[6] / s, r[7] / s);
        *reinterpret_cast<uint2*>(const_cast<uint8_t*>(a.k) + at) = o;
      } else {
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(a.k)) + at) = make_uint4(
            pack_bf16_pair_rne(r[0], r[1]), pack_bf16_pair_rne(r[2], r[3]), pack_bf16_pair_rne(r[4], r[5]),
            pack_bf16_pair_rne(r[6], r[7]));
      }
    }
  }
  if (!there || n_vt) return;
  const uint16_t* v = p.v + static_cast<size_t>(t) * p.kv_ld;
  for (uint32_t i = tid; i < a.n_kv * HD; i += threads) {  // one token: one transposed column
    const uint32_t h = i / HD, d = i % HD;
    const size_t at = ((page0 + h) * HD + d) * pg + off;
    if constexpr (F8)
      const_cast<uint8_t*>(a.v)[at] =
          static_cast<uint8_t>(pack_e4m3x4(bf16_to_f32(v[i]) / a.v_scale[h], 0.0f, 0.0f, 0.0f));
    else
      reinterpret_cast<uint16_t*>(const_cast<uint8_t*>(a.v))[at] = v[i];
  }
}

// ---------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------
// Order-preserving image of a weight: larger weight, larger key; -0 as +0; NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return w != w ? 0u : ((u >> 31) ? ~u : (u | 0x80000000u));
}

constexpr uint32_t EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64u, EV_KEYS = 16, EV_BINS = 2048;

// Exclusive scan over the workgroup, in thread order; s_w: EV_WAVES words, other
// ones than the scan before (whose readers the barrier here does not hold back).
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t* s_w, uint32_t lane, uint32_t wave, uint32_t& total) {
  const uint32_t incl = wave_scan_u32(v);
  if (lane == 63u) s_w[wave] = incl;
  __syncthreads();
  const uint32_t w = lane < EV_WAVES ? s_w[lane] : 0u, ws = wave_scan_u32(w);
  total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ws), EV_WAVES - 1u));
  const uint32_t before = wave ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ws), static_cast<int>(wave) - 1)) : 0u;
  return before + incl - v;
}

// One workgroup per (sequence, kv head). The entries' weights lie in registers,
// up to 16 consecutive ones a thread (16,384 entries at once; longer sequences
// pass through in segments, again for each step). Three steps of 11, 11 and 10
// bits find the K-th largest key of the entries between the first and the last
// ones: counts by digit in LDS, then a scan from the top. Attention weights
// spread over many powers of two, so the top digit (sign, exponent, two mantissa
// bits) has few lanes at one counter. One more scan, of the sure entries and the
// ties together, gives the kept ones' places; they are listed in LDS, so that the
// stores are whole lines (from each thread by itself they took a third of the
// kernel). The third step falls away where the second one's bin is kept whole.
// Bound by latency and one CU's issue rate: 9.1 us for 8,192 entries (2.0 until
// the weights are there, 3.5 for two steps, 2.1 for the places and stores),
// 16 for 96 rows of up to 16,003, 91 for one sequence of 100,003 (seven segments,
// three or four times each).
__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(Paged a, Weight w, Weight wd, uint32_t sinks,
                                                                 uint32_t recent, uint32_t budget,
                                                                 int32_t* __restrict__ kept,
                                                                 int32_t* __restrict__ new_len) {
  constexpr uint32_t SEG = EV_KEYS * EV_THREADS;
  __shared__ __attribute__((aligned(16))) uint32_t s_mem[SEG / 2u];
  uint32_t(*const s_hist)[EV_BINS] = reinterpret_cast<uint32_t(*)[EV_BINS]>(s_mem);  // one a step, cleared together
  uint16_t* const s_list = reinterpret_cast<uint16_t*>(s_mem);                       // afterwards: a segment's kept entries
  static_assert(SEG / 2u >= 3u * EV_BINS && SEG <= 65536u, "the counters, and places in 16 bits");
  __shared__ uint32_t s_w[2][EV_WAVES];
  __shared__ uint32_t s_pick[3];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6);
  const uint32_t b = blockIdx.x / a.n_kv, h = blockIdx.x % a.n_kv;
  const uint32_t n = uniform(paged_len(a, b)), now = umin(n, budget);
  const int64_t slot = weight_slot(w, b), dslot = weight_slot(wd, b);
  if (tid == 0u) {
    if (paged_len_bad(a, b) || (n > 0u && (slot < 0 || dslot < 0))) paged_flag(a.status);  // (a padded batch needs no slots)
    if (h == 0u) new_len[b] = static_cast<int32_t>(now);
  }
  const float* src = w.w + (static_cast<size_t>(max(slot, int64_t(0))) * a.n_kv + h) * w.ld;
  float* dst = wd.w + (static_cast<size_t>(max(dslot, int64_t(0))) * a.n_kv + h) * wd.ld;
  int32_t* kp = kept + (static_cast<size_t>(b) * a.n_kv + h) * budget;
  for (uint32_t e = now + tid; e < budget; e += EV_THREADS) kp[e] = -1;
  // entries a thread holds of a segment: a multiple of 4, so its loads can be 16 bytes
  const uint32_t per = umin(EV_KEYS, ((n + EV_THREADS - 1u) / EV_THREADS + 3u) & ~3u), seg = per * EV_THREADS;
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0u;
  const uint32_t lo = n > budget ? sinks : n, hi = n > budget ? n - recent : n;  // the candidates [lo, hi)
  auto range_bits = [&](uint32_t j0, uint32_t from, uint32_t end) {  // of the `per` entries from j0, those in [from, end)
    return below_bits(j0, end) & ~below_bits(j0, from) & ((1u << per) - 1u);
  };
  uint32_t key[EV_KEYS], mid = 0u;  // mid: bits of the thread's candidates
  uint32_t held = 0xffffffffu;
  auto load = [&](uint32_t s0) __attribute__((always_inline)) {  // the segment from entry s0
    if (held == s0) return;  // uniform
    held = s0;
    const uint32_t j0 = s0 + per * tid;
    float wt[EV_KEYS];
#pragma unroll
    for (uint32_t i = 0; i < EV_KEYS; i += 4u) {
      if (i >= per) break;  // uniform
      if (slot < 0) {
        wt[i] = wt[i + 1] = wt[i + 2] = wt[i + 3] = 0.0f;
      } else if (vec && j0 + i + 4u <= n) {
        const float4 v = *reinterpret_cast<const float4*>(src + j0 + i);
        wt[i] = v.x;
        wt[i + 1] = v.y;
        wt[i + 2] = v.z;
        wt[i + 3] = v.w;
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) wt[i + j] = j0 + i + j < n ? src[j0 + i + j] : 0.0f;
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < EV_KEYS; ++i) {
      if (i >= per) break;  // uniform
      key[i] = weight_key(wt[i]);
    }
    mid = range_bits(j0, lo, hi);
  };
  uint32_t want = n > budget ? budget - sinks - recent : 0u;  // < hi - lo
  uint32_t thr = 0xffffffffu, ties = 0u;  // kept: key > thr, and the first `ties` with key == thr
  if (want > 0u) {  // uniform
    uint32_t prefix = 0u;
    bool exact = false;  // all entries of the last digit's bin are kept (usual after two steps)
    load(0u);
    for (uint32_t i = tid; i < 3u * EV_BINS; i += EV_THREADS) s_mem[i] = 0u;
    __syncthreads();
#pragma unroll
    for (uint32_t step = 0; step < 3; ++step) {
      if (exact) break;  // uniform
      const uint32_t shift = step == 0u ? 21u : step == 1u ? 10u : 0u, bits = step == 2u ? 10u : 11u;
      for (uint32_t s0 = 0; s0 < n; s0 += seg) {
        load(s0);
#pragma unroll
        for (uint32_t i = 0; i < EV_KEYS; ++i) {
          if (i >= per) break;  // uniform
          if ((mid >> i & 1u) && (step == 0u || ((key[i] ^ prefix) >> (shift + bits)) == 0u))
            atomicAdd(&s_hist[step][(key[i] >> shift) & ((1u << bits) - 1u)], 1u);
        }
      }
      __syncthreads();
      // thread t looks at bins top - 2 t and top - 2 t - 1: the one where the count from the top reaches `want`
      const uint32_t top = EV_BINS - 1u - 2u * tid, c1 = s_hist[step][top], c0 = s_hist[step][top - 1u];
      uint32_t total;
      const uint32_t above = group_scan(c0 + c1, s_w[step & 1u], lane, wave, total);
      if (above < want && above + c0 + c1 >= want) {  // one thread
        const bool first = above + c1 >= want;
        s_pick[0] = first ? top : top - 1u;
        s_pick[1] = want - above - (first ? 0u : c1);
        s_pick[2] = first ? c1 : c0;
      }
      __syncthreads();
      prefix |= s_pick[0] << shift;
      want = s_pick[1];  // (written again only behind the next step's barriers)
      exact = s_pick[2] == want && prefix > 0u;
    }
    thr = exact ? prefix - 1u : prefix;
    ties = exact ? 0u : want;
  }
  uint32_t sure_at = 0u, tie_at = 0u;  // of the segments before
  for (uint32_t s0 = 0, par = 1u; s0 < n; s0 += seg, par ^= 1u) {
    load(s0);
    const uint32_t j0 = s0 + per * tid;
    uint32_t tie = 0u, above = 0u;  // bits of the thread's entries
#pragma unroll
    for (uint32_t i = 0; i < EV_KEYS; ++i) {
      if (i >= per) break;  // uniform
      tie |= key[i] == thr ? 1u << i : 0u;
      above |= key[i] > thr ? 1u << i : 0u;
    }
    tie &= ties ? mid : 0u;
    uint32_t keep = (range_bits(j0, 0u, n) & ~mid) | (above & mid);
    uint32_t sums;
    const uint32_t before = group_scan(static_cast<uint32_t>(__popc(keep)) << 16 | static_cast<uint32_t>(__popc(tie)),
                                       s_w[par], lane, wave, sums);
    uint32_t rank = tie_at + (before & 0xffffu);  // of the thread's first tie
    const uint32_t ties_before = umin(tie_at, ties);
    uint32_t x = (before >> 16) + umin(rank, ties) - ties_before;  // place among the segment's kept entries
#pragma unroll
    for (uint32_t i = 0; i < EV_KEYS; ++i) {
      if (i >= per) break;  // uniform
      if (tie >> i & 1u) keep |= rank++ < ties ? 1u << i : 0u;
      if (keep >> i & 1u) s_list[x++] = static_cast<uint16_t>(per * tid + i);
    }
    const uint32_t first = sure_at + ties_before;
    sure_at += sums >> 16;
    tie_at += sums & 0xffffu;
    const uint32_t count = sure_at + umin(tie_at, ties) - first;
    __syncthreads();
    for (uint32_t i = tid; i < count; i += EV_THREADS) {
      const uint32_t j = s0 + s_list[i], e = first + i;
      if (e >= budget) break;
      kp[e] = static_cast<int32_t>(j);
      if (dslot >= 0) dst[e] = slot >= 0 ? src[j] : 0.0f;
    }
  }
}

// GE (64, or 16 where that leaves CUs idle) kept entries of one (sequence, kv
// head) a workgroup. Keys: rows of 16-byte
// chunks. Values: a wave takes 64 dims (32 where a head has 64), a dim a lane,
// of 16 entries: the entries are the wave's, so their pages are scalar bases,
// neighbours in one 16-byte chunk share a load, all loads are in flight before
// the first is taken apart, and a lane writes 16 consecutive entries of its row.
// A transposed value page is read whole as soon as one of its entries is kept
// (an entry's dims lie a row apart).
template <uint32_t HD, bool F8, uint32_t GE>
__global__ void __launch_bounds__(256) evict_copy_kernel(Paged a, const int32_t* __restrict__ dst_pages,
                                                         uint32_t dst_max_pages, uint32_t budget,
                                                         const int32_t* __restrict__ kept) {
  typedef typename std::conditional<F8, uint8_t, uint16_t>::type T;
  constexpr uint32_t SZ = sizeof(T), CH = HD * SZ / 16u;  // 16-byte chunks of a key row
  __shared__ int32_t s_src[GE], s_dst[GE];                // pages of both sides, -1: none
  __shared__ uint32_t s_so[GE];                           // entries in the source pages
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), groups = (budget + GE - 1u) / GE;
  const uint32_t gi = blockIdx.x % groups, bh = blockIdx.x / groups, b = bh / a.n_kv, h = bh % a.n_kv;
  const uint32_t mask = (1u << a.lp) - 1u, e0 = GE * gi;
  if (tid < GE) {
    const uint32_t e = e0 + tid;
    const int32_t j = e < budget ? kept[static_cast<size_t>(bh) * budget + e] : -1;
    int32_t s = -1, d = -1;
    if (j >= 0) {
      bool ok;
      const uint32_t sp = paged_id(a, b, static_cast<uint32_t>(j), ok);
      if (ok) s = static_cast<int32_t>(sp);
      const uint32_t dp = static_cast<uint32_t>(dst_pages[static_cast<size_t>(b) * dst_max_pages + (e >> a.lp)]);
      if (dp < a.n_pages) d = static_cast<int32_t>(dp);
      if (s < 0 || d < 0) paged_flag(a.status);
    }
    s_so[tid] = static_cast<uint32_t>(j) & mask;
    s_src[tid] = s;
    s_dst[tid] = d;
  }
  __syncthreads();
  uint8_t* const kb = const_cast<uint8_t*>(a.k);
  constexpr uint32_t KN = (GE * CH + 255u) / 256u;  // a thread's chunks: all read before the first is written
  uint4 kx[KN];
#pragma unroll
  for (uint32_t i = 0; i < KN; ++i) {
    const uint32_t t = tid + 256u * i, e = t / CH % GE, c = t % CH;
    const size_t row = ((static_cast<size_t>(max(s_src[e], 0)) * a.n_kv + h) << a.lp) + s_so[e];
    kx[i] = *reinterpret_cast<const uint4*>(kb + row * (HD * SZ) + 16u * c);
    if (s_src[e] < 0) kx[i] = make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (uint32_t i = 0; i < KN; ++i) {
    const uint32_t t = tid + 256u * i, e = t / CH % GE, c = t % CH;
    if ((GE * CH % 256u == 0u || t < GE * CH) && s_dst[e] >= 0) {
      const size_t row = ((static_cast<size_t>(s_dst[e]) * a.n_kv + h) << a.lp) + ((e0 + e) & mask);
      *reinterpret_cast<uint4*>(kb + row * (HD * SZ) + 16u * c) = kx[i];
    }
  }
  constexpr uint32_t DW = HD / 64u;  // waves across the dims
  const T* vs = reinterpret_cast<const T*>(a.v);
  T* vd = reinterpret_cast<T*>(const_cast<uint8_t*>(a.v));
  const uint32_t d = 64u * (wave % DW) + lane;
  for (uint32_t q = wave / DW; q < GE / 16u; q += 4u / DW) {  // 16 entries, of one destination page
    const int32_t dp = static_cast<int32_t>(uniform(static_cast<uint32_t>(s_dst[16u * q])));
    if (dp < 0) continue;  // uniform: no page, or behind the last entry
    T x[16];
    uint32_t cnt = 0;  // entries of the destination page
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
      cnt += uniform(static_cast<uint32_t>(s_dst[16u * q + i])) == static_cast<uint32_t>(dp) ? 1u : 0u;
    if constexpr (GE == 16u) {  // few entries: a load each, the shortest way (both kernels 15.4 us against 17.1; of many 137 against 118)
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const int32_t sp = static_cast<int32_t>(uniform(static_cast<uint32_t>(s_src[16u * q + i])));
        // (a page that is not there reads page 0)
        const T* row = vs + ((static_cast<size_t>(max(sp, 0)) * a.n_kv + h) * HD << a.lp) + uniform(s_so[16u * q + i]);
        x[i] = row[d << a.lp];
        if (sp < 0) x[i] = 0;  // uniform
      }
    } else {
      // one load for the entries of one 16-byte chunk (CE neighbours of a row)
      constexpr uint32_t CE = 16u / SZ;
      u32x4_v ch[16];
      uint32_t fresh = 0;  // entries that begin another chunk
      uint32_t ps = 0xffffffffu, pc = 0u;
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const uint32_t e = 16u * q + i, sp = uniform(static_cast<uint32_t>(s_src[e])), c = uniform(s_so[e]) / CE;
        if (i == 0u || sp != ps || c != pc) {  // uniform
          fresh |= 1u << i;
          // (a page that is not there reads page 0)
          const T* row = vs + ((static_cast<size_t>(static_cast<int32_t>(sp) < 0 ? 0u : sp) * a.n_kv + h) * HD << a.lp) + CE * c;
          ch[i] = *reinterpret_cast<const u32x4_v*>(row + (d << a.lp));
          if (static_cast<int32_t>(sp) < 0) ch[i] = u32x4_v{0u, 0u, 0u, 0u};
        }
        ps = sp;
        pc = c;
      }
      u32x4_v cur = ch[0];
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        if (i && (fresh >> i & 1u)) cur = ch[i];  // uniform
        const uint32_t k = uniform(s_so[16u * q + i]) % CE, byte = k * SZ % 8u;  // its bytes in the chunk's half
        const uint32_t pick = SZ == 2u ? (0x0c0c0000u | (byte + 1u) << 8 | byte) : (0x0c0c0c00u | byte);
        const uint32_t lo = __builtin_amdgcn_perm(cur.y, cur.x, pick), hi = __builtin_amdgcn_perm(cur.w, cur.z, pick);
        x[i] = static_cast<T>(k * SZ < 8u ? lo : hi);
      }
    }
    T* to = vd + ((static_cast<size_t>(dp) * a.n_kv + h) * HD << a.lp) + (static_cast<size_t>(d) << a.lp) + ((e0 + 16u * q) & mask);
    if (cnt == 16u) {  // uniform
      uint32_t o[4 * SZ];
#pragma unroll
      for (uint32_t i = 0; i < 4 * SZ; ++i) {
        if constexpr (F8)
          o[i] = x[4 * i] | x[4 * i + 1] << 8 | x[4 * i + 2] << 16 | static_cast<uint32_t>(x[4 * i + 3]) << 24;
        else
          o[i] = x[2 * i] | static_cast<uint32_t>(x[2 * i + 1]) << 16;
      }
#pragma unroll
      for (uint32_t i = 0; i < SZ; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i)
        if (i < cnt) to[i] = x[i];
    }
  }
}

// Waves a token row: four, or one where rows fill the chip and it goes at most five
// times round the heads, as the chain to a row's entry and position then runs in
// fewer waves (6,000 rows of 36 heads of 64: 32.0 us with four, 18.0 with one, of 14
// heads 28.2 and 11.9; of 36 heads of 128, nine times round, one gains nothing).
uint32_t prep_waves(uint32_t hd, uint32_t heads, uint32_t rows) { return heads * hd <= 2560u && rows >= 1024u ? 1u : 4u; }

template <uint32_t HD, bool F8>
int launch_prep(obs_ctx* ctx, const Paged& a, const PrepArgs& p, const Weight& w, uint32_t n_vt, uint32_t grid, uint32_t waves) {
  if (waves == 1u)
    OBS_LAUNCH(ctx, "attn_prep_paged", prep_paged_kernel<HD, F8, 1><<<grid, 256, 0, ctx->stream>>>(a, p, w, n_vt));
  else
    OBS_LAUNCH(ctx, "attn_prep_paged", prep_paged_kernel<HD, F8, 4><<<grid, 256, 0, ctx->stream>>>(a, p, w, n_vt));
  return OBS_OK;
}

// copies: workgroups with 64 entries each.
template <uint32_t HD, bool F8>
int launch_copy(obs_ctx* ctx, const Paged& a, const int32_t* dst_pages, uint32_t dst_max_pages, uint32_t budget,
                const int32_t* kept, uint64_t copies) {
  // below two workgroups a CU (a few sequences): 16 entries each, one sequence of 2,048 kept entries 15.4 us against 19.9
  if (copies < 512u) {
    const uint32_t grid = a.n_seqs * a.n_kv * ((budget + 15u) / 16u);
    OBS_LAUNCH(ctx, "kv_evict_copy",
               evict_copy_kernel<HD, F8, 16><<<grid, 256, 0, ctx->stream>>>(a, dst_pages, dst_max_pages, budget, kept));
  } else {
    const uint32_t grid = static_cast<uint32_t>(copies);
    OBS_LAUNCH(ctx, "kv_evict_copy",
               evict_copy_kernel<HD, F8, 64><<<grid, 256, 0, ctx->stream>>>(a, dst_pages, dst_max_pages, budget, kept));
  }
  return OBS_OK;
}

}  // namespace

namespace obs {

int paged_status(obs_ctx* ctx) {
  uint32_t st = 0;
  OBS_HIP_TRY(ctx, hipStreamSynchronize(ctx->stream));
  OBS_HIP_TRY(ctx, hipMemcpy(&st, ctx->status_dev + CTX_ST_PAGED, sizeof st, hipMemcpyDeviceToHost));
  if (!st) return OBS_OK;
  OBS_HIP_TRY(ctx, hipMemset(ctx->status_dev + CTX_ST_PAGED, 0, sizeof st));
  OBS_HIP_TRY(ctx, hipDeviceSynchronize());
  return set_error(ctx, OBS_E_INVALID, "paged cache: a page id, length or slot in device memory was out of range");
}

int check_paged(obs_ctx* ctx, const char* who, const obs_paged_kv* kv, const obs_paged_seqs* s, bool pointers) {
  if (!kv || !s) return set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
  if (kv->dtype != OBS_KV_BF16 && kv->dtype != OBS_KV_E4M3)
    return set_error(ctx, OBS_E_INVALID, "%s: dtype must be OBS_KV_BF16 or OBS_KV_E4M3 (got %d)", who, kv->dtype);
  if (pointers) {
    if (!kv->k_pages || !kv->v_pages || !s->pages || !s->len || (kv->dtype == OBS_KV_E4M3 && (!kv->k_scale || !kv->v_scale)))
      return set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
    if (!aligned(kv->k_pages, 16) || !aligned(kv->v_pages, 16))
      return set_error(ctx, OBS_E_ALIGN, "%s: the pages must be 16-byte aligned", who);
  }
  if ((kv->head_dim != 64u && kv->head_dim != 128u) || kv->page < 16u || kv->page > 256u || (kv->page & (kv->page - 1u)) ||
      kv->n_kv == 0 || kv->n_kv > 1024u || kv->n_pages == 0 || kv->n_pages > 0x7fffffffu ||
      static_cast<uint64_t>(kv->n_pages) * kv->n_kv > 0xffffffffull)
    return set_error(ctx, OBS_E_SHAPE,
                     "%s: head_dim must be 64 or 128, page a power of two in [16, 256], n_kv in [1, 1024], n_pages in "
                     "[1, 2^31) with n_pages * n_kv below 2^32 (got %u, %u, %u, %u)", who, kv->head_dim, kv->page, kv->n_kv, kv->n_pages);
  if (s->n_seqs > PAGED_MAX_SEQS || s->max_pages == 0 ||
      static_cast<uint64_t>(s->max_pages) * kv->page > PAGED_MAX_ENTRIES || s->n_rows > (1u << 24))
    return set_error(ctx, OBS_E_SHAPE,
                     "%s: at most %u sequences, 1 to 2^30 / page pages each and 2^24 token rows (got %u, %u, %u)", who,
                     PAGED_MAX_SEQS, s->n_seqs, s->max_pages, s->n_rows);
  return OBS_OK;
}

int check_heads(obs_ctx* ctx, const char* who, uint32_t n_heads, uint32_t n_kv) {
  if (n_heads == 0 || n_heads % n_kv != 0 || n_heads / n_kv > 16u)
    return set_error(ctx, OBS_E_SHAPE, "%s: n_heads must be a multiple of n_kv with at most 16 per kv head (got %u, %u)",
                     who, n_heads, n_kv);
  return OBS_OK;
}

int check_grid(obs_ctx* ctx, const char* who, uint64_t workgroups, uint32_t threads) {
  if (workgroups > 0xffffffffull / threads)
    return set_error(ctx, OBS_E_SHAPE, "%s: too much for one call (%llu workgroups of %u)", who,
                     static_cast<unsigned long long>(workgroups), threads);
  return OBS_OK;
}

int check_weight(obs_ctx* ctx, const char* who, const obs_kv_weight* w, uint64_t entries, bool pointers) {
  if (pointers && !w->w) return set_error(ctx, OBS_E_INVALID, "%s: null weight", who);
  if (pointers && !aligned(w->w, 4)) return set_error(ctx, OBS_E_ALIGN, "%s: weight must be 4-byte aligned", who);
  if (w->n_slots == 0 || w->n_slots > 0x7fffffffu || w->ld < entries)
    return set_error(ctx, OBS_E_SHAPE, "%s: weight needs slots and rows of at least %llu entries (got %u, %u)", who,
                     static_cast<unsigned long long>(entries), w->n_slots, w->ld);
  return OBS_OK;
}

}  // namespace obs

extern "C" {

int obs_attn_prep_paged(obs_ctx* ctx, const obs_paged_kv* kv, const obs_paged_seqs* seqs, const obs_kv_weight* weight,
                        const uint16_t* q, const uint16_t* k, const uint16_t* v, const uint16_t* q_norm,
                        const uint16_t* k_norm, uint16_t* q_out, uint32_t n_heads, float eps, float theta,
                        const int32_t* pos, uint32_t rope_len, uint32_t q_ld, uint32_t kv_ld, uint32_t q_out_ld) {
  if (!ctx) return OBS_E_INVALID;
  const char* who = "obs_attn_prep_paged";
  int rc = obs::check_paged(ctx, who, kv, seqs, true);
  if (rc == OBS_OK) rc = obs::check_heads(ctx, who, n_heads, kv->n_kv);
  if (rc == OBS_OK && weight) rc = obs::check_weight(ctx, who, weight, static_cast<uint64_t>(seqs->max_pages) * kv->page, true);
  if (rc != OBS_OK) return rc;
  if (!q || !k || !v || !q_norm || !k_norm || !q_out) return obs::set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
  if (!seqs->row && seqs->n_rows != seqs->n_seqs)
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: without row, n_rows must be n_seqs (got %u, %u)", who, seqs->n_rows, seqs->n_seqs);
  const uint32_t hd = kv->head_dim;
  q_ld = q_ld ? q_ld : n_heads * hd;
  kv_ld = kv_ld ? kv_ld : kv->n_kv * hd;
  q_out_ld = q_out_ld ? q_out_ld : n_heads * hd;
  if (q_ld < n_heads * hd || kv_ld < kv->n_kv * hd || q_out_ld < n_heads * hd || q_ld % 8u || kv_ld % 8u || q_out_ld % 8u)
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: row strides %u, %u, %u must be multiples of 8 and hold a row", who, q_ld, kv_ld, q_out_ld);
  if (q_out == q && q_out_ld != q_ld)
    return obs::set_error(ctx, OBS_E_INVALID, "%s: q_out may be q only with the same row stride", who);
  if (!obs::aligned(q, 16) || !obs::aligned(k, 16) || !obs::aligned(v, 16) || !obs::aligned(q_norm, 16) ||
      !obs::aligned(k_norm, 16) || !obs::aligned(q_out, 16))
    return obs::set_error(ctx, OBS_E_ALIGN, "%s: q, k, v, the norm weights and q_out must be 16-byte aligned", who);
  if (rope_len == 0 || rope_len > (1u << 24))
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: rope_len must be in [1, 2^24] (got %u)", who, rope_len);
  if (seqs->n_rows == 0 || seqs->n_seqs == 0) return OBS_OK;
  const uint32_t n_vt = seqs->row ? kv->n_kv * ((seqs->n_rows + PREP_TILE - 1u) / PREP_TILE) : 0u;
  const uint32_t waves = prep_waves(hd, n_heads + kv->n_kv, seqs->n_rows);
  const uint32_t grid = n_vt + (waves == 1u ? (seqs->n_rows + 3u) / 4u : seqs->n_rows);
  rc = obs::check_grid(ctx, who, grid, 256u);
  if (rc != OBS_OK) return rc;
  obs::DeviceGuard guard(ctx);
  PrepArgs p{q, k, v, q_norm, k_norm, q_out, pos, nullptr, n_heads, rope_len, q_ld, kv_ld, q_out_ld, eps};
  rc = obs::ensure_rope_table(ctx, theta, rope_len, &p.rope, obs::ROPE_EXACT_FROM, obs::rope_rows(rope_len));
  if (rc != OBS_OK) return rc;
  const Paged a = obs::paged_args(ctx, kv, seqs);
  const Weight w = obs::weight_args(weight);
  const bool f8 = kv->dtype == OBS_KV_E4M3;
  if (hd == 128u)
    return f8 ? launch_prep<128, true>(ctx, a, p, w, n_vt, grid, waves) : launch_prep<128, false>(ctx, a, p, w, n_vt, grid, waves);
  return f8 ? launch_prep<64, true>(ctx, a, p, w, n_vt, grid, waves) : launch_prep<64, false>(ctx, a, p, w, n_vt, grid, waves);
}

int obs_kv_evict(obs_ctx* ctx, const obs_paged_kv* kv, const obs_paged_seqs* seqs, const obs_kv_weight* weight,
                 const int32_t* dst_pages, uint32_t dst_max_pages, const obs_kv_weight* dst_weight, uint32_t sinks,
                 uint32_t recent, uint32_t budget, int32_t* kept, int32_t* new_len) {
  if (!ctx) return OBS_E_INVALID;
  const char* who = "obs_kv_evict";
  int rc = obs::check_paged(ctx, who, kv, seqs, true);
  if (rc != OBS_OK) return rc;
  if (!weight || !dst_weight || !dst_pages || !kept || !new_len)
    return obs::set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
  rc = obs::check_weight(ctx, who, weight, static_cast<uint64_t>(seqs->max_pages) * kv->page, true);
  if (rc == OBS_OK) rc = obs::check_weight(ctx, who, dst_weight, budget, true);
  if (rc != OBS_OK) return rc;
  if (budget == 0 || static_cast<uint64_t>(sinks) + recent > budget || dst_max_pages == 0 ||
      static_cast<uint64_t>(dst_max_pages) * kv->page > obs::PAGED_MAX_ENTRIES ||
      budget > static_cast<uint64_t>(dst_max_pages) * kv->page)
    return obs::set_error(ctx, OBS_E_SHAPE,
                          "%s: sinks + recent <= budget <= dst_max_pages * page, at most 2^30 entries (got %u + %u, %u, %u pages)",
                          who, sinks, recent, budget, dst_max_pages);
  if (seqs->n_seqs == 0) return OBS_OK;
  const uint64_t copies = static_cast<uint64_t>(seqs->n_seqs) * kv->n_kv * ((budget + 63u) / 64u);
  // arrays that the call's workgroups read while others write them
  if (new_len == seqs->len || dst_pages == seqs->pages || (weight->w == dst_weight->w && weight->slot == dst_weight->slot))
    return obs::set_error(ctx, OBS_E_INVALID, "%s: new_len, the destination's pages and its weight rows must not be the source's", who);
  rc = obs::check_grid(ctx, who, copies, 256u);
  if (rc == OBS_OK) rc = obs::check_grid(ctx, who, static_cast<uint64_t>(seqs->n_seqs) * kv->n_kv, EV_THREADS);
  if (rc != OBS_OK) return rc;
  obs::DeviceGuard guard(ctx);
  const Paged a = obs::paged_args(ctx, kv, seqs);
  OBS_LAUNCH(ctx, "kv_evict_select", evict_select_kernel<<<seqs->n_seqs * kv->n_kv, EV_THREADS, 0, ctx->stream>>>(
                                         a, obs::weight_args(weight), obs::weight_args(dst_weight), sinks, recent, budget,
                                         kept, new_len));
  const bool f8 = kv->dtype == OBS_KV_E4M3, d128 = kv->head_dim == 128u;
  return d128 ? (f8 ? launch_copy<128, true>(ctx, a, dst_pages, dst_max_pages, budget, kept, copies)
                    : launch_copy<128, false>(ctx, a, dst_pages, dst_max_pages, budget, kept, copies))
              : (f8 ? launch_copy<64, true>(ctx, a, dst_pages, dst_max_pages, budget, kept, copies)
                    : launch_copy<64, false>(ctx, a, dst_pages, dst_max_pages, budget, kept, copies));
}

}  // extern "C"
