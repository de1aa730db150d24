// obs_logprobs.hip — log probabilities of given tokens, the entropy and the most
// likely alternatives, from logits (obs_token_logprobs) or from hidden rows and the
// 4-bit output matrix (obs_lm_logprobs).
//
// With m the largest of a set of logits, s = sum e and w = sum e (x - m),
// e = exp(x - m), sets are joined by taking s and w to the larger maximum
// (w' = f (w + s (m - m')), f = exp(m - m')). Of the whole row
//   log p(t) = x_t - m - log s,   entropy = log s - w / s,
// sums of one sign each. The k largest of a row lie in the k tiles with the largest
// maxima, ties to the lower tile, so only those are looked through.
#include <algorithm>

#include "obs_internal.hpp"
#include "obs_paged.hpp"

namespace {
using namespace obsd;

constexpr float LOG2E = 1.44269504088896341f, FAR = -1.0e4f;
constexpr uint32_t MAX_TOP = 64;

struct Stat {
  float m = NEG_INF, s = 0.0f, w = 0.0f;
};
__device__ __forceinline__ Stat stat_of(const float4& v) {
  Stat r;
  r.m = v.x;
  r.s = v.y;
  r.w = v.z;
  return r;
}
// s and w taken to the maximum m (a set without a logit above -inf has s = w = 0; NaN stays)
__device__ __forceinline__ void stat_to(Stat& a, float m) {
  const float d = fmaxf(a.m - (m == NEG_INF ? 0.0f : m), FAR), f = __builtin_amdgcn_exp2f(d * LOG2E);
  a.w = f * __builtin_fmaf(a.s, d, a.w);
  a.s *= f;
  a.m = m;
}
template <uint32_t N>
__device__ __forceinline__ void stat_add(Stat& a, const float (&x)[N], float top) {  // top: the largest of x
  const float m = fmaxf(a.m, top);
  if (m > a.m) stat_to(a, m);
  const float mu = a.m == NEG_INF ? 0.0f : a.m;
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    const float d = x[i] - mu, e = __builtin_amdgcn_exp2f(d * LOG2E);
    a.s += e;
    a.w = __builtin_fmaf(e, fmaxf(d, FAR), a.w);
  }
}
// Over the workgroup's four waves; s_st: four words each of three, another barrier before their next use.
__device__ __forceinline__ Stat stat_group(Stat a, float (*s_st)[4], uint32_t lane, uint32_t wave) {
  stat_to(a, wave_max_f32(a.m));
  const float s = wave_sum_asc(a.s), w = wave_sum_asc(a.w);
  if (lane == 0u) {
    s_st[0][wave] = a.m;
    s_st[1][wave] = s;
    s_st[2][wave] = w;
  }
  __syncthreads();
  Stat r;
  r.m = fmaxf(fmaxf(s_st[0][0], s_st[0][1]), fmaxf(s_st[0][2], s_st[0][3]));
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    Stat b;
    b.m = s_st[0][i];
    b.s = s_st[1][i];
    b.w = s_st[2][i];
    stat_to(b, r.m);
    r.s += b.s;
    r.w += b.w;
  }
  return r;
}

// ---------------------------------------------------------------------------
// The k largest of what a wave sees
// ---------------------------------------------------------------------------
// A key is a value's order-preserving image above the complement of its index:
// larger value, larger key; of equal ones the lower index. Lane i holds the i-th
// largest key met (0: none yet); `edge` keeps out what cannot be among the k.
__device__ __forceinline__ uint64_t top_key(float v, uint32_t index) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // (-0 as +0)
  return static_cast<uint64_t>((u >> 31) ? ~u : u | 0x80000000u) << 32 | ~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((u >> 31) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~static_cast<uint32_t>(key); }
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, uint32_t l) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), static_cast<int>(l)));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), static_cast<int>(l)));
  return static_cast<uint64_t>(hi) << 32 | lo;
}
constexpr uint64_t NONE_KEY = 0x007fffffffffffffull;  // of -inf (0x007fffff in the upper word): nothing at or below it counts
struct Top {
  uint64_t key = 0u, edge = NONE_KEY;
  // every lane offers a key (0: none)
  __device__ __forceinline__ void offer(uint64_t c, uint32_t k, uint32_t lane) {
    for (;;) {
      const uint64_t mask = __ballot(c > edge);
      if (!mask) break;  // uniform
      const uint32_t l = static_cast<uint32_t>(__builtin_ctzll(mask));
      const uint64_t x = lane_u64(c, l);
      const uint32_t at = static_cast<uint32_t>(__popcll(__ballot(key > x)));
      const uint32_t lo = static_cast<uint32_t>(__shfl_up(static_cast<int>(key), 1)),
                     hi = static_cast<uint32_t>(__shfl_up(static_cast<int>(key >> 32), 1));
      key = lane > at ? (static_cast<uint64_t>(hi) << 32 | lo) : lane == at ? x : key;
      const uint64_t last = lane_u64(key, k - 1u);
      edge = last > edge ? last : edge;
      if (lane == l) c = 0u;
    }
  }
};

// ---------------------------------------------------------------------------
// Logits
// ---------------------------------------------------------------------------
// A workgroup takes one part of a row, a wave a step of 1,024 logits at once: their sums,
// and the maxima of its four tiles, of 16 lanes each (a wave's whole maximum of every
// load cost 7 of 57 us for 777 rows in bf16). One pass; bound by the reading.
template <bool BF16>
struct Logits {
  static constexpr uint32_t LOAD = BF16 ? 512u : 256u, PER = LOAD / 64u, STEP = 1024u, N = STEP / LOAD;
  // PER logits from i on (behind the row's end: -inf)
  static __device__ __forceinline__ void load(const void* row, uint32_t i, uint32_t n, bool vec, float* x) {
    if constexpr (BF16) {
      const uint16_t* p = static_cast<const uint16_t*>(row) + i;
      if (vec && i + PER <= n) {
        const uint4 v = load_stream(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
          x[2 * j] = bf16lo(w[j]);
          x[2 * j + 1] = bf16hi(w[j]);
        }
      } else {
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) x[j] = i + j < n ? bf16_to_f32(p[j]) : NEG_INF;
      }
    } else {
      const float* p = static_cast<const float*>(row) + i;
      if (vec && i + PER <= n) {
        const uint4 v = load_stream(p);
        x[0] = __uint_as_float(v.x);
        x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z);
        x[3] = __uint_as_float(v.w);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) x[j] = i + j < n ? p[j] : NEG_INF;
      }
    }
  }
};

template <bool BF16>
__global__ void __launch_bounds__(256) logits_part_kernel(const uint8_t* __restrict__ logits, size_t row_bytes,
                                                          uint32_t vocab, uint32_t parts, float4* __restrict__ stat,
                                                          float* __restrict__ tmax, uint32_t tiles) {
  typedef Logits<BF16> L;
  __shared__ float s_st[3][4];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6);
  const uint32_t t = blockIdx.x / parts, part = blockIdx.x % parts;
  const uint8_t* row = logits + t * row_bytes;
  const bool vec = (reinterpret_cast<uintptr_t>(row) & 15u) == 0u;
  const uint32_t steps = (vocab + L::STEP - 1u) / L::STEP;
  Stat a;
  for (uint32_t s = 4u * part + wave; s < steps; s += 4u * parts) {
    float x[L::N][L::PER];
#pragma unroll
    for (uint32_t j = 0; j < L::N; ++j) L::load(row, s * L::STEP + j * L::LOAD + L::PER * lane, vocab, vec, x[j]);
    float top[L::N];
#pragma unroll
    for (uint32_t j = 0; j < L::N; ++j) {
      top[j] = x[j][0];
#pragma unroll
      for (uint32_t i = 1; i < L::PER; ++i) top[j] = fmaxf(top[j], x[j][i]);
    }
#pragma unroll
    for (uint32_t j = 0; j < L::N; ++j) stat_add<L::PER>(a, x[j], top[j]);
    if (tmax) {  // uniform
      float m = top[0];
#pragma unroll
      for (uint32_t j = 1; j < L::N; ++j) m = fmaxf(m, top[j]);
      m = fmaxf(m, dpp_f32<DPP_XOR1>(m));
      m = fmaxf(m, dpp_f32<DPP_XOR2>(m));
      m = fmaxf(m, dpp_f32<DPP_HALF_MIRROR>(m));
      m = fmaxf(m, dpp_f32<DPP_MIRROR>(m));
      // (of NaN alone: -inf)
      if (lane % 16u == 0u) tmax[static_cast<size_t>(t) * tiles + 4u * s + lane / 16u] = fmaxf(m, NEG_INF);
    }
  }
  const Stat r = stat_group(a, s_st, lane, wave);
  if (tid == 0u) stat[static_cast<size_t>(t) * parts + part] = make_float4(r.m, r.s, r.w, 0.0f);
}

struct JoinArgs {
  const float4* stat;  // [rows][n_stat]
  const float* tmax;   // maximum of tile i of row t at [t * tiles + i] * tstride
  const uint8_t* logits;
  const float* xt;  // the tokens' logits, or null: from the logits
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_lp;
  size_t row_bytes;
  uint32_t n_stat, tiles, tstride, vocab, k;
};

// The largest value with its lower 16 bits clear that at least k of the lanes' keys
// reach: two scalar instructions a bit. Keys: f32_order above the least int.
__device__ __forceinline__ float lanes_edge(float own, uint32_t k) {
  const uint32_t key = static_cast<uint32_t>(f32_order(own)) ^ 0x80000000u;
  uint32_t e = 0u;
#pragma unroll
  for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1) {
    const uint32_t at = e | bit;
    if (static_cast<uint32_t>(__popcll(__ballot(key >= at))) >= k) e = at;  // uniform
  }
  // (nothing below -inf)
  return e < 0x00800000u ? NEG_INF : f32_unorder(static_cast<int>(e ^ 0x80000000u));
}

// A workgroup a row: the parts' sums joined, then the k largest. Of the tiles: what k
// lanes of a wave reach with their own maxima keeps out all but a few, which are listed in
// LDS and ranked by counting; the same of the k tiles' logits. Where more are listed than
// there is room for (equal values in masses), a wave takes them one by one. The code runs
// once, so its length counts. (A wave's lists from the start took 21 us a row of 2,374
// tiles at k = 5; ranks of all 256 threads' maxima, and every load's listing unrolled, 17.)
// TILE: tile i has the TILE logits from TILE i on; 0: logits_part_kernel's, 256 logits
// each, four interleaved in a step. Steps are in order, so with the k-th tile come those of
// its step, the next three at most.
template <bool BF16, uint32_t TILE>
__global__ void __launch_bounds__(256) logprobs_join_kernel(JoinArgs p) {
  constexpr uint32_t CAP = 1024, SUBS = TILE ? 1u : 4u, PER = TILE == 64u ? 1u : 4u;
  __shared__ float s_st[3][4];
  __shared__ uint32_t s_tile[MAX_TOP + 4u], s_n[2];
  __shared__ uint64_t s_list[CAP];
  __shared__ float s_edge[5];  // of the waves; the k-th tile's maximum
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), t = blockIdx.x, k = p.k;
  const uint8_t* row = p.logits + t * p.row_bytes;
  const float* tm = p.tmax + static_cast<size_t>(t) * p.tiles * p.tstride;
  const float4* st = p.stat + static_cast<size_t>(t) * p.n_stat;
  auto logit = [&](uint32_t i) __attribute__((always_inline)) {
    return BF16 ? bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[i]) : reinterpret_cast<const float*>(row)[i];
  };
  // the token's logit is on its way before anything waits
  const int32_t tok = p.tokens ? p.tokens[t] : -1;
  const bool there = tok >= 0 && static_cast<uint32_t>(tok) < p.vocab;
  const float own_x = !there ? 0.0f : p.xt ? p.xt[t] : logit(static_cast<uint32_t>(tok));
  // v[i]: maximum of tile i0 + 256 i + tid, -inf behind the last
  auto maxima = [&](uint32_t i0, float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = tm[static_cast<size_t>(umin(i0 + 256u * i + tid, p.tiles - 1u)) * p.tstride];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = i0 + 256u * i + tid < p.tiles ? v[i] : NEG_INF;
  };
  float first[8], own = NEG_INF;  // of the first 2,048 tiles
  if (k) {
    if (tid < 2u) s_n[tid] = 0u;
    if (tid < MAX_TOP + 4u) s_tile[tid] = 0xffffffffu;
    if (tid == 0u) s_edge[4] = NEG_INF;
    maxima(0u, first);
  }
  Stat a;
  for (uint32_t i0 = 0; i0 < p.n_stat; i0 += 1024u) {
    float4 v[4];
    float m = a.m;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t at = i0 + 256u * i + tid;
      v[i] = st[umin(at, p.n_stat - 1u)];
      if (at >= p.n_stat) v[i] = make_float4(NEG_INF, 0.0f, 0.0f, 0.0f);
      m = fmaxf(m, v[i].x);
    }
    stat_to(a, m);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      Stat b = stat_of(v[i]);
      stat_to(b, m);
      a.s += b.s;
      a.w += b.w;
    }
  }
  if (k) {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) own = fmaxf(own, first[i]);
    for (uint32_t i = 2048u + tid; i < p.tiles; i += 256u) own = fmaxf(own, tm[static_cast<size_t>(i) * p.tstride]);
    const float e = lanes_edge(own, k);
    if (lane == 0u) s_edge[wave] = e;
  }
  const Stat r = stat_group(a, s_st, lane, wave);  // a barrier: the waves' edges are there
  const float ls = logf(r.s);
  const bool none = r.m == NEG_INF && r.s == 0.0f;  // no logit above -inf
  if (tid == 0u) {
    if (p.entropy) p.entropy[t] = none ? 0.0f : ls - r.w / r.s;
    if (p.logprob) p.logprob[t] = !there ? 0.0f : none ? NEG_INF : (own_x - r.m) - ls;
  }
  if (!k) return;
  auto list = [&](uint32_t which, uint64_t key) __attribute__((always_inline)) {
    const uint32_t at = atomicAdd(&s_n[which], 1u);
    if (at < CAP) s_list[at] = key;
  };
  // the place of a listed key among the n: how many are larger
  auto place = [&](uint64_t key, uint32_t n) __attribute__((always_inline)) {
    uint32_t above = 0;
    for (uint32_t i = 0; i < n; i += 4u)
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) above += s_list[i + j] > key && i + j < n;  // (read before it is known to count: in flight together)
    return above;
  };
  const float edge = fmaxf(fmaxf(s_edge[0], s_edge[1]), fmaxf(s_edge[2], s_edge[3]));
  for (uint32_t i0 = 0;;) {
    uint32_t mask = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) mask |= first[i] >= edge && first[i] > NEG_INF ? 1u << i : 0u;
    while (mask) {  // few
      const uint32_t i = static_cast<uint32_t>(__builtin_ctz(mask)), at = i0 + 256u * i + tid;
      mask &= mask - 1u;
      list(0u, top_key(tm[static_cast<size_t>(at) * p.tstride], at));
    }
    i0 += 2048u;
    if (i0 >= p.tiles) break;
    maxima(i0, first);
  }
  __syncthreads();
  uint32_t n = uniform(s_n[0]);
  const bool room = n <= CAP;  // else s_tile holds steps
  if (room) {  // uniform
    for (uint32_t i = tid; i < n; i += 256u) {
      const uint64_t key = s_list[i];
      const uint32_t at = place(key, n);
      if (at < k + SUBS - 1u) s_tile[at] = key_index(key);
      if (at == k - 1u) s_edge[4] = key_value(key);
    }
  } else if (wave == 0u) {
    Top top;
    for (uint32_t i0 = 0; i0 < p.tiles; i0 += 64u * SUBS) {
      const uint32_t at = i0 + SUBS * lane;
      float m = NEG_INF;
#pragma unroll
      for (uint32_t i = 0; i < SUBS; ++i) m = fmaxf(m, at + i < p.tiles ? tm[static_cast<size_t>(at + i) * p.tstride] : NEG_INF);
      top.offer(at < p.tiles ? top_key(m, at / SUBS) : 0u, k, lane);
    }
    if (lane < k && top.key) s_tile[lane] = key_index(top.key);
    if (lane == k - 1u && top.key) s_edge[4] = key_value(top.key);
  }
  __syncthreads();
  // the logits of those tiles that are as large as the last one's maximum: a wave takes
  // every fourth tile, four of them in flight
  const float low = s_edge[4];
  const bool vec = (reinterpret_cast<uintptr_t>(row) & 15u) == 0u;
  auto first_of = [&](uint32_t tile) __attribute__((always_inline)) {  // of the lane's PER logits
    if constexpr (TILE)
      return tile * TILE + PER * lane;
    else if constexpr (BF16)
      return tile / 4u * 1024u + 512u * (lane / 32u) + 128u * (tile % 4u) + 4u * (lane % 32u);
    else
      return tile / 4u * 1024u + 256u * (lane / 16u) + 64u * (tile % 4u) + 4u * (lane % 16u);
  };
  const uint32_t rows = room ? k + SUBS - 1u : k * SUBS;
  auto tile_of = [&](uint32_t j) __attribute__((always_inline)) {
    if (room) return s_tile[umin(j, MAX_TOP + 3u)];
    const uint32_t step = s_tile[umin(j / SUBS, MAX_TOP - 1u)];
    return step == 0xffffffffu ? step : step * SUBS + j % SUBS;
  };
  auto load = [&](uint32_t j, float (&x)[PER]) __attribute__((always_inline)) {  // -inf where there is none
    const uint32_t tile = uniform(tile_of(j)), v = first_of(tile);
    const bool is = j < rows && tile != 0xffffffffu;  // uniform
    if (PER == 4u && is && vec && v + PER <= p.vocab) {
      if constexpr (BF16) {
        const uint2 w = *reinterpret_cast<const uint2*>(row + 2u * static_cast<size_t>(v));
        const uint32_t u[2] = {w.x, w.y};
#pragma unroll
        for (uint32_t e = 0; e < PER; ++e) x[e] = e & 1u ? bf16hi(u[e / 2u]) : bf16lo(u[e / 2u]);
      } else {
        const float4 w = *reinterpret_cast<const float4*>(row + 4u * static_cast<size_t>(v));
        const float u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (uint32_t e = 0; e < PER; ++e) x[e] = u[e];
      }
    } else {
#pragma unroll
      for (uint32_t e = 0; e < PER; ++e) x[e] = is && v + e < p.vocab ? logit(v + e) : NEG_INF;
    }
  };
  for (uint32_t j0 = wave; j0 < rows; j0 += 16u) {
    float x[4][PER];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) load(j0 + 4u * i, x[i]);
    uint32_t mask = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
      for (uint32_t e = 0; e < PER; ++e) mask |= x[i][e] >= low && x[i][e] > NEG_INF ? 1u << (PER * i + e) : 0u;  // (not NaN)
    while (mask) {  // few
      const uint32_t b = static_cast<uint32_t>(__builtin_ctz(mask)), v = first_of(tile_of(j0 + 4u * (b / PER))) + b % PER;
      mask &= mask - 1u;
      list(1u, top_key(logit(v), v));
    }
  }
  __syncthreads();
  n = uniform(s_n[1]);
  auto write = [&](uint32_t at, uint64_t key) __attribute__((always_inline)) {
    p.top_ids[static_cast<size_t>(t) * k + at] = key ? static_cast<int32_t>(key_index(key)) : -1;
    p.top_lp[static_cast<size_t>(t) * k + at] = key ? (key_value(key) - r.m) - ls : NEG_INF;
  };
  if (n <= CAP) {  // uniform
    for (uint32_t i = tid; i < n; i += 256u) {
      const uint64_t key = s_list[i];
      const uint32_t at = place(key, n);
      if (at < k) write(at, key);
    }
    if (tid >= n && tid < k) write(tid, 0u);  // fewer than k
  } else if (wave == 0u) {
    Top top;
    for (uint32_t j = 0; j < rows; ++j) {
      float x[PER];
      load(j, x);
      const uint32_t v = first_of(tile_of(j));
#pragma unroll
      for (uint32_t e = 0; e < PER; ++e) top.offer(x[e] > NEG_INF ? top_key(x[e], v + e) : 0u, k, lane);
    }
    if (lane < k) write(lane, top.key);
  }
}

// ---------------------------------------------------------------------------
// Hidden rows and the 4-bit output matrix
// ---------------------------------------------------------------------------
// logit[t][v] = sum_g s (sum q x) + b (sum x) over the groups g of 64 columns, s and b
// of (v, g). The products take the nibbles themselves, exact, in products of tokens x
// vocabulary, so that a lane has one vocabulary row and the scale is one factor of its sums
// over a group, in fp32: no weight is rounded.
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16_v;
constexpr uint32_t LM_COLS = 256, LM_FEW_COLS = 64;  // vocabulary rows of a workgroup

// Eight nibbles as 16 + q in bf16, columns 0, 4, 1, 5, 2, 6, 3, 7.
__device__ __forceinline__ bf16x8_v lm_weights(uint32_t w) {
  return __builtin_bit_cast(bf16x8_v, u32x4_v{q4_bf16<0>(w), q4_bf16<2>(w), q4_bf16<1>(w), q4_bf16<3>(w)});
}
// Eight columns in that order.
__device__ __forceinline__ u32x4_v lm_order(const uint4& v) {
  return u32x4_v{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                 __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
}
__device__ __forceinline__ float sum8(const uint4& v) {
  return ((bf16lo(v.x) + bf16hi(v.x)) + (bf16lo(v.y) + bf16hi(v.y))) + ((bf16lo(v.z) + bf16hi(v.z)) + (bf16lo(v.w) + bf16hi(v.w)));
}
__device__ __forceinline__ float sum_of_8_lanes(float v) {
  v += dpp_f32<DPP_XOR1>(v);
  v += dpp_f32<DPP_XOR2>(v);
  return v + dpp_f32<DPP_HALF_MIRROR>(v);
}

struct LmArgs {
  const uint16_t* x;
  const uint32_t* w;
  const uint16_t* s;
  const uint16_t* b;
  const int32_t* tokens;
  float* xt;
  float4* stat;   // [T][tiles]
  float* logits;  // [T][ld], or null
  uint32_t T, in, vocab, tiles, ld;
};

// The token of row t, or one that is no column's (padding).
__device__ __forceinline__ uint32_t lm_token(const LmArgs& p, uint32_t t) {
  const uint32_t tok = static_cast<uint32_t>(p.tokens[t]);
  return tok < p.vocab ? tok : 0xffffffffu;
}
// A row's COLS logits x of the workgroup, L lanes of N each (the lane's V-th at column
// STEP (V / 4) + 4 lane + V % 4): their sums, and the logits where they are wanted. L is 8
// or 16 lanes of a row of lanes; `first` is the row's first.
template <uint32_t COLS, uint32_t L, uint32_t N>
__device__ __forceinline__ void lm_sums(const LmArgs& p, float (&x)[N], uint32_t t, uint32_t v0, uint32_t part, bool is) {
  static_assert(L * N == COLS && (L == 8u || L == 16u), "whole rows");
  constexpr uint32_t STEP = 4u * L;
  const uint32_t at = v0 + 4u * part;
  if (p.logits) {  // uniform
#pragma unroll
    for (uint32_t i = 0; i < N; i += 4)
      if (is && at + STEP * (i / 4u) < p.ld)
        *reinterpret_cast<float4*>(p.logits + static_cast<size_t>(t) * p.ld + at + STEP * (i / 4u)) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  }
  if (v0 + COLS > p.vocab) {  // uniform: the last columns
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[i] = at + STEP * (i / 4u) + i % 4u < p.vocab ? x[i] : NEG_INF;
  }
  float m = x[0];
#pragma unroll
  for (uint32_t i = 1; i < N; ++i) m = fmaxf(m, x[i]);
  auto over = [&](float v, auto op) __attribute__((always_inline)) {
    v = op(v, dpp_f32<DPP_XOR1>(v));
    v = op(v, dpp_f32<DPP_XOR2>(v));
    v = op(v, dpp_f32<DPP_HALF_MIRROR>(v));
    return L == 16u ? op(v, dpp_f32<DPP_MIRROR>(v)) : v;
  };
  m = fmaxf(over(m, [](float a, float b) { return fmaxf(a, b); }), NEG_INF);  // (of NaN alone: -inf)
  Stat a;
  a.m = m;
  stat_add<N>(a, x, m);
  const float s = over(a.s, [](float a, float b) { return a + b; }), w = over(a.w, [](float a, float b) { return a + b; });
  if (is && part == 0u) p.stat[static_cast<size_t>(t) * p.tiles + v0 / COLS] = make_float4(m, s, w, 0.0f);
}

// Up to 16 NT tokens: the weights go through once and bound the call. A workgroup a CU
// takes 64 vocabulary rows after another, each of its eight waves a slice of 256 columns
// (of more than 2,048 several in turn), with the next weights in flight beside this one's
// products; the slices meet in LDS. (Workgroups of one tile each loaded, computed and
// ended together: 75 to 94 us a token in three shapes of them.) A lane (col = lane % 16, q
// = lane / 16) of a product (v_mfma_f32_16x16x32_bf16) loads 16 bytes of its row, the four
// 64, two groups; a swap of the wave's halves gives each lane 8 bytes of either (of the
// group's 32, those from 16 (q % 2) + 8 (q / 2) on). The sums over a group's columns are a
// product with ones. HELD: a wave has one slice, whose rows of x stay in registers.
template <uint32_t NT, bool HELD>
__global__ void __launch_bounds__(512, 2) lm_few_kernel(LmArgs p) {
  constexpr uint32_t RT = 16u * NT, OROW = LM_FEW_COLS + 4u, WAVES = 8;
  __shared__ __attribute__((aligned(16))) float s_out[2][WAVES][RT][OROW];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), col = lane & 15u, q = lane >> 4;
  const uint32_t groups = p.in / 64u, slices = p.in / 256u, per = HELD ? 1u : (slices + WAVES - 1u) / WAVES;
  uint32_t xoff[NT];
#pragma unroll
  for (uint32_t m = 0; m < NT; ++m) xoff[m] = umin(16u * m + col, p.T - 1u) * (2u * p.in) + 64u * (q & 1u) + 32u * (q >> 1);  // (behind the last token it again)
  const u32x4_v one4 = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  const bf16x8_v ones = __builtin_bit_cast(bf16x8_v, one4);
  const f32x4_v zero = {0.0f, 0.0f, 0.0f, 0.0f};
  auto load_x = [&](uint32_t slice, uint32_t g, uint32_t s, uint32_t m) __attribute__((always_inline)) {
    const uint8_t* xb = reinterpret_cast<const uint8_t*>(p.x) + 512u * slice;
    return __builtin_bit_cast(bf16x8_v, lm_order(*reinterpret_cast<const uint4*>(xb + (xoff[m] + 128u * g + 16u * s))));
  };
  bf16x8_v xh[HELD ? 4 : 1][2][NT];
  if constexpr (HELD) {
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g)
#pragma unroll
      for (uint32_t s = 0; s < 2; ++s)
#pragma unroll
        for (uint32_t m = 0; m < NT; ++m) xh[g][s][m] = load_x(umin(wave, slices - 1u), g, s, m);
  }
  struct Rows {
    u32x4_v w[4][2];     // two groups each
    u32x2_v s[4], b[4];  // of four
  } cur, nxt;
  // a slice behind the last one reads the last one's, without use
  auto load_w = [&](Rows& k, uint32_t tile, uint32_t slice) __attribute__((always_inline)) {
    const uint32_t v0 = tile * LM_FEW_COLS;
    const uint8_t *wb = reinterpret_cast<const uint8_t*>(p.w) + static_cast<size_t>(v0) * (p.in / 2u) + 128u * slice,
                  *sb = reinterpret_cast<const uint8_t*>(p.s) + static_cast<size_t>(v0) * (2u * groups) + 8u * slice,
                  *bb = reinterpret_cast<const uint8_t*>(p.b) + static_cast<size_t>(v0) * (2u * groups) + 8u * slice;
#pragma unroll
    for (uint32_t n = 0; n < 4; ++n) {
      const uint32_t r = umin(16u * n + col, p.vocab - 1u - v0);  // (behind the last row it again)
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) k.w[n][h] = *reinterpret_cast<const u32x4_v*>(wb + (r * (p.in / 2u) + 16u * q + 64u * h));
      k.s[n] = *reinterpret_cast<const u32x2_v*>(sb + r * (2u * groups));
      k.b[n] = *reinterpret_cast<const u32x2_v*>(bb + r * (2u * groups));
    }
  };
  f32x4_v acc[4][NT] = {};
  uint32_t tile = blockIdx.x, j = 0, buf = 0;
  // the token of the thread's row, as below
  const uint32_t token = p.tokens && tid / 16u < p.T ? lm_token(p, tid / 16u) : 0xffffffffu;
  load_w(cur, tile, umin(wave, slices - 1u));
  for (;;) {
    // the next slice of these rows, or the first of the next ones
    const bool end = j + 1u == per;
    const uint32_t ntile = end ? tile + gridDim.x : tile, nj = end ? 0u : j + 1u;
    load_w(nxt, umin(ntile, p.tiles - 1u), umin(wave + WAVES * nj, slices - 1u));
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t slice = wave + WAVES * j;
    if (slice < slices) {  // uniform
#pragma unroll
      for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
          for (uint32_t i = 0; i < 2; ++i) {
            const auto r = __builtin_amdgcn_permlane32_swap(cur.w[n][h][i], cur.w[n][h][i + 2u], false, false);
            cur.w[n][h][i] = r[0];
            cur.w[n][h][i + 2u] = r[1];
          }
#pragma unroll
      for (uint32_t g = 0; g < 4; ++g) {
        bf16x8_v xa[2][NT];
        f32x4_v xs[NT];
#pragma unroll
        for (uint32_t s = 0; s < 2; ++s)
#pragma unroll
          for (uint32_t m = 0; m < NT; ++m) {
            if constexpr (HELD)
              xa[s][m] = xh[g][s][m];
            else
              xa[s][m] = load_x(slice, g, s, m);
            xs[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa[s][m], ones, s ? xs[m] : zero, 0, 0, 0);
          }
#pragma unroll
        for (uint32_t n = 0; n < 4; ++n) {
          f32x4_v y[NT];
#pragma unroll
          for (uint32_t s = 0; s < 2; ++s) {
            const bf16x8_v wb = lm_weights(cur.w[n][g / 2u][2u * (g & 1u) + s]);
#pragma unroll
            for (uint32_t m = 0; m < NT; ++m) y[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xa[s][m], wb, s ? y[m] : zero, 0, 0, 0);
          }
          const uint32_t sw = cur.s[n][g / 2u], bw = cur.b[n][g / 2u];
          const float sc = g & 1u ? bf16hi(sw) : bf16lo(sw), off = __builtin_fmaf(sc, -16.0f, g & 1u ? bf16hi(bw) : bf16lo(bw));
#pragma unroll
          for (uint32_t m = 0; m < NT; ++m)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) acc[n][m][i] = __builtin_fmaf(sc, y[m][i], __builtin_fmaf(off, xs[m][i], acc[n][m][i]));
        }
      }
    }
    if (end) {  // uniform
#pragma unroll
      for (uint32_t n = 0; n < 4; ++n)
#pragma unroll
        for (uint32_t m = 0; m < NT; ++m) {
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) s_out[buf][wave][16u * m + 4u * q + i][16u * n + col] = acc[n][m][i];
          acc[n][m] = zero;
        }
      __syncthreads();
      // sixteen threads a row, four columns each
      const uint32_t t = tid / 16u, part = tid % 16u;
      if (t / 4u < (p.T + 3u) / 4u) {  // whole waves
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) {
          const f32x4_v v = *reinterpret_cast<const f32x4_v*>(&s_out[buf][w][umin(t, RT - 1u)][4u * part]);
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) x[i] += v[i];
        }
        const uint32_t k = token - tile * LM_FEW_COLS - 4u * part;  // (a token behind the last one is no row's)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
          if (k == i) p.xt[t] = x[i];
        lm_sums<LM_FEW_COLS, 16>(p, x, t, tile * LM_FEW_COLS, part, t < p.T);
      }
      buf ^= 1u;  // (read again two tiles on, behind a barrier that its readers pass first)
      if (ntile >= p.tiles) break;
    }
    tile = ntile;
    j = nj;
    cur = nxt;
  }
}

// Many tokens: bound by the matrix units, beside which the weights come apart and one
// product a sum and group goes with the scale, in the vector unit. A nibble masked in
// place at bits 3:0 (7:4) of a half word is the fp16 number q 2^-24 (q 2^-20), subnormal,
// which the products (v_mfma_f32_32x32x16_f16) take as it is: five instructions for eight
// nibbles, and no offset. The rows are brought into fp16 by a power of two a row, its
// largest to 2^14: exact from 2^-29 of that on (the columns of upper nibbles 2^-25, as they
// get a sixteenth), off by 2^-38 of it below. (Products of 8-bit numbers, of which a bf16 x
// has two, would need masks alone, but they drop what lies 2^-13 below the largest of eight
// products.)
//
// First the rows in the order of the products' operands, [tile of 32 MT rows][group][32
// rows][step][lane] 16 bytes, each row's factor back, and the sums of every group in three
// bf16 parts (24 bits), which meet the biases in products of their own at the end of a
// tile. A wave takes a row.
constexpr uint32_t LM_SUMS = 3;
template <uint32_t MT>
__global__ void __launch_bounds__(512) lm_rows_kernel(const uint16_t* __restrict__ x, uint32_t T, uint32_t in, uint8_t* __restrict__ xp,
                                                      float* __restrict__ xf, uint8_t* __restrict__ xs) {
  const uint32_t lane = threadIdx.x & 63u, t = blockIdx.x * 8u + uniform(threadIdx.x >> 6), mt = t / 32u, r = t % 32u;
  const uint32_t groups = in / 64u, gpad = (groups + 15u) & ~15u, chunks = in / 8u;  // a multiple of 64
  const uint16_t* row = x + static_cast<size_t>(t < T ? t : 0u) * in;
  uint32_t most = 0u;
  for (uint32_t c = lane; c < chunks; c += 64u) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + 8u * c);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) most = max(most, max(w[e] & 0x7fffu, w[e] >> 16 & 0x7fffu));
  }
  const uint32_t ex = max(wave_max_u31(most) >> 7, 15u);
  const float up = __uint_as_float((268u - ex) << 23);
  if (lane == 0u) xf[t] = t < T ? __uint_as_float((ex - 2u) << 23) : 0.0f;  // back, and 2^12 of the nibbles' 2^24
  for (uint32_t c = lane; c < gpad * 8u; c += 64u) {
    const uint32_t g = c / 8u;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (t < T && g < groups) v = *reinterpret_cast<const uint4*>(row + 8u * c);
    const float sum = sum_of_8_lanes(sum8(v));
    if (g < groups) {
      // half c / 4 % 2, step c % 4: columns 0, 4 | 1, 5 | 2, 6 | 3, 7 of the eight
      auto pair = [&](float a, float b, float f) __attribute__((always_inline)) {
        return __builtin_bit_cast(uint32_t, f16x2_of(a * f, b * f));
      };
      const float od = up * 0.0625f;
      *reinterpret_cast<uint4*>(xp + 16u * (((static_cast<size_t>(mt / MT) * groups + g) * MT + mt % MT) * 256u + c % 4u * 64u + 32u * (c / 4u % 2u) + r)) =
          make_uint4(pair(bf16lo(v.x), bf16lo(v.z), up), pair(bf16hi(v.x), bf16hi(v.z), od), pair(bf16lo(v.y), bf16lo(v.w), up),
                     pair(bf16hi(v.y), bf16hi(v.w), od));
    }
    if (c % 8u == 0u) {
      float rest = sum;
#pragma unroll
      for (uint32_t k = 0; k < LM_SUMS; ++k) {
        const uint16_t part = f32_to_bf16(rest);
        rest -= bf16_to_f32(part);
        // steps of 16 groups, eight a lane's half
        reinterpret_cast<uint16_t*>(xs + 16u * ((static_cast<size_t>(mt) * LM_SUMS * (gpad / 16u) + k * (gpad / 16u) + g / 16u) * 64u +
                                                32u * (g / 8u % 2u) + r))[g % 8u] = part;
      }
    }
  }
}

// 32 MT tokens x 256 vocabulary rows a workgroup, 64 a wave; two workgroups a CU.
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
template <uint32_t MT>
__global__ void __launch_bounds__(256, 2) lm_many_kernel(LmArgs p, const uint8_t* __restrict__ xp, const float* __restrict__ xf,
                                                         const uint8_t* __restrict__ xs, uint32_t ttiles) {
  constexpr uint32_t XB = MT * 4096u, OROW = LM_COLS + 8u, OB = 32u * OROW * 4u;  // bytes of a group's rows; of 32 rows of logits
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[2u * XB > OB ? 2u * XB : OB];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6), col = lane & 31u, half = lane >> 5;
  // an XCD (blockIdx.x % 8) takes all token tiles of one column tile after another: its weights stay in its L2
  const uint32_t at = blockIdx.x / 8u, vt = at / ttiles * 8u + blockIdx.x % 8u, tt = at % ttiles;
  if (vt >= p.tiles) return;  // uniform
  const uint32_t v0 = vt * LM_COLS, groups = p.in / 64u, gpad = (groups + 15u) & ~15u;
  // scalar bases and 32-bit offsets of the lane's rows
  const uint8_t *wb0 = reinterpret_cast<const uint8_t*>(p.w) + static_cast<size_t>(v0) * (p.in / 2u),
                *sb0 = reinterpret_cast<const uint8_t*>(p.s) + static_cast<size_t>(v0) * (2u * groups),
                *bb0 = reinterpret_cast<const uint8_t*>(p.b) + static_cast<size_t>(v0) * (2u * groups);
  uint32_t woff[2], soff[2];
#pragma unroll
  for (uint32_t n = 0; n < 2; ++n) {
    const uint32_t r = umin(v0 + 64u * wave + 32u * n + col, p.vocab - 1u) - v0;  // (behind the last row it again)
    woff[n] = r * (p.in / 2u) + 16u * half;
    soff[n] = r * (2u * groups);
  }
  const uint8_t* xg = xp + static_cast<size_t>(tt) * groups * XB;
  u32x4_v xr[MT];
  auto load_x = [&](uint32_t g) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < MT; ++i) xr[i] = *reinterpret_cast<const u32x4_v*>(xg + static_cast<size_t>(g) * XB + (16u * tid + 4096u * i));
  };
  auto store_x = [&](uint32_t buf) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < MT; ++i) *reinterpret_cast<u32x4_v*>(s_mem + buf * XB + 16u * tid + 4096u * i) = xr[i];
  };
  f32x16_v acc[MT][2];
#pragma unroll
  for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n) acc[m][n] = f32x16_v{};
  u32x4_v wr[2];  // a group ahead
  uint32_t sr[2];
  auto load_w = [&](uint32_t g) __attribute__((always_inline)) {
    const uint32_t gc = umin(g, groups - 1u);
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n) {
      wr[n] = *reinterpret_cast<const u32x4_v*>(wb0 + 32u * gc + woff[n]);
      sr[n] = *reinterpret_cast<const uint16_t*>(sb0 + 2u * gc + soff[n]);
    }
  };
  load_x(0u);
  load_w(0u);
  store_x(0u);
  __syncthreads();
  auto step = [&](uint32_t g, uint32_t slot) __attribute__((always_inline)) {
    f16x8_v xa[4], wb[2][4];
    float sc[2];
    auto load_a = [&](uint32_t m, uint32_t s) __attribute__((always_inline)) {
      xa[s] = *reinterpret_cast<const f16x8_v*>(s_mem + slot * XB + 16u * ((m * 4u + s) * 64u + lane));
    };
#pragma unroll
    for (uint32_t s = 0; s < 4; ++s) load_a(0u, s);
    load_x(umin(g + 1u, groups - 1u));
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n) {
      sc[n] = __uint_as_float(sr[n] << 16) * 4096.0f;
#pragma unroll
      for (uint32_t s = 0; s < 4; ++s) {
        const uint32_t w = wr[n][s], w8 = w >> 8;
        wb[n][s] = __builtin_bit_cast(f16x8_v, u32x4_v{w & 0x000f000fu, w & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u});
      }
    }
    load_w(g + 1u);
    __builtin_amdgcn_sched_barrier(0);
    // Products of one 32 x 32 tile, each beside a quarter of the sums of the tile before and,
    // with the last use of its rows, the read of the next ones: left to itself the compiler
    // puts a tile's sums behind its products, and the two units take turns.
    f32x16_v y[2];
    const f32x16_v zero = {};
#pragma unroll
    for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
      for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s) {
          y[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xa[s], wb[n][s], s ? y[n] : zero, 0, 0, 0);
          if (n == 1u && m + 1u < MT) load_a(m + 1u, s);
          if (m || n) {
            const uint32_t pm = n ? m : m - 1u, pn = 1u - n;
#pragma unroll
            for (uint32_t i = 4u * s; i < 4u * s + 4u; ++i) acc[pm][pn][i] = __builtin_fmaf(sc[pn], y[pn][i], acc[pm][pn][i]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) acc[MT - 1u][1][i] = __builtin_fmaf(sc[1], y[1][i], acc[MT - 1u][1][i]);
    store_x(slot ^ 1u);
    __syncthreads();
  };
  for (uint32_t g = 0; g < groups; g += 2u) {  // groups is a multiple of 8
    step(g, 0u);
    step(g + 1u, 1u);
  }
  uint32_t token[MT];  // of the rows that the thread has below
#pragma unroll
  for (uint32_t m = 0; m < MT; ++m) {
    const uint32_t t = 32u * (tt * MT + m) + tid / 8u;
    token[m] = p.tokens && t < p.T ? lm_token(p, t) : 0xffffffffu;
  }
  // the rows' factors back (and 2^12 of the nibbles'), then the groups' sums with the biases
#pragma unroll
  for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
    for (uint32_t i = 0; i < 16; i += 4) {
      const f32x4_v f = *reinterpret_cast<const f32x4_v*>(xf + 32u * (tt * MT + m) + 2u * i + 4u * half);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) {
        acc[m][0][i + e] *= f[e];
        acc[m][1][i + e] *= f[e];
      }
    }
  const uint32_t steps = gpad / 16u;
  for (uint32_t s = 0; s < steps; ++s) {
    const uint32_t g = 16u * s + 8u * half;
    bf16x8_v bb[2];
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n) {
      u32x4_v v = *reinterpret_cast<const u32x4_v*>(bb0 + (soff[n] + 2u * umin(g, groups - 8u)));
      if (g >= groups) v = u32x4_v{0u, 0u, 0u, 0u};
      bb[n] = __builtin_bit_cast(bf16x8_v, v);
    }
#pragma unroll
    for (uint32_t k = 0; k < LM_SUMS; ++k)
#pragma unroll
      for (uint32_t m = 0; m < MT; ++m) {
        const bf16x8_v xa = *reinterpret_cast<const bf16x8_v*>(
            xs + 16u * (((static_cast<size_t>(tt) * MT + m) * LM_SUMS * steps + k * steps + s) * 64u + lane));
#pragma unroll
        for (uint32_t n = 0; n < 2; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xa, bb[n], acc[m][n], 0, 0, 0);
      }
  }
  // 32 rows at a time through LDS, eight threads a row. (A wave a row, one after another, took
  // as long as the products: 740 us of 1,470 for 2,000 tokens.)
  float(*const s_out)[OROW] = reinterpret_cast<float(*)[OROW]>(s_mem);
  const uint32_t orow = tid / 8u, part = tid % 8u;
#pragma unroll
  for (uint32_t m = 0; m < MT; ++m) {
    if (m) __syncthreads();
#pragma unroll
    for (uint32_t n = 0; n < 2; ++n)
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) s_out[8u * (i / 4u) + 4u * half + i % 4u][64u * wave + 32u * n + col] = acc[m][n][i];
    __syncthreads();
    const uint32_t t = 32u * (tt * MT + m) + orow, k = token[m] - v0;
    if (part == 0u && k < LM_COLS) p.xt[t] = s_out[orow][k];
    float x[32];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const f32x4_v v = *reinterpret_cast<const f32x4_v*>(&s_out[orow][32u * i + 4u * part]);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) x[4 * i + e] = v[e];
    }
    lm_sums<LM_COLS, 8>(p, x, t, v0, part, t < p.T);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
using obs::up256;

struct LogitsPlan {
  uint32_t parts, tiles;
  size_t stat, tmax;  // bytes
};
LogitsPlan logits_plan(uint32_t T, uint32_t vocab, uint32_t k) {
  LogitsPlan d{};
  // eight workgroups a CU, of 4,096 logits at least
  d.parts = std::max(1u, std::min((2047u + T) / std::max(T, 1u), (vocab + 4095u) / 4096u));
  d.tiles = (vocab + 1023u) / 1024u * 4u;
  d.stat = up256(static_cast<size_t>(T) * d.parts * sizeof(float4));
  d.tmax = k ? up256(static_cast<size_t>(T) * d.tiles * sizeof(float)) : 0u;
  return d;
}

constexpr uint32_t LM_FEW = 32;
struct LmPlan {
  uint32_t rows, mt, tiles, ld;  // token rows of a pass, 32-row blocks of a workgroup
  size_t stat, xt, logits, xp, xf, xs;
  size_t all() const { return stat + xt + logits + xp + xf + xs; }
};
LmPlan lm_plan(uint32_t T, uint32_t in, uint32_t vocab, uint32_t k) {
  LmPlan d{};
  const uint32_t cols = T <= LM_FEW ? LM_FEW_COLS : LM_COLS;
  d.tiles = (vocab + cols - 1u) / cols;
  d.ld = (vocab + 3u) & ~3u;
  // the logits of a pass where alternatives are wanted, and its sums, are of a bounded size
  d.rows = T <= LM_FEW ? T : std::min(T, k ? 256u : 4096u);
  d.mt = d.rows <= 64u ? 2u : 3u;
  const size_t groups = in / 64u, gpad = (groups + 15u) & ~size_t(15), blocks = (d.rows + 32u * d.mt - 1u) / (32u * d.mt) * d.mt;
  d.stat = up256(static_cast<size_t>(d.rows) * d.tiles * sizeof(float4));
  d.xt = up256(static_cast<size_t>(d.rows) * sizeof(float));
  d.logits = k ? up256(static_cast<size_t>(d.rows) * d.ld * sizeof(float)) : 0u;
  if (T > LM_FEW) {
    d.xp = up256(blocks * 64u * in);
    d.xf = up256(blocks * 32u * sizeof(float));
    d.xs = up256(blocks * LM_SUMS * gpad * 64u);
  }
  return d;
}

int check_outputs(obs_ctx* ctx, const char* who, const int32_t* tokens, const float* logprob, uint32_t top_k, uint32_t vocab,
                  const int32_t* top_ids, const float* top_logprobs) {
  if ((tokens == nullptr) != (logprob == nullptr) || (top_k && (!top_ids || !top_logprobs)))
    return obs::set_error(ctx, OBS_E_INVALID, "%s: tokens and logprob go together, and top_k needs its outputs", who);
  if (top_k > MAX_TOP || top_k > vocab)
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: top_k must be at most %u and at most vocab (got %u)", who, MAX_TOP, top_k);
  return OBS_OK;
}
int check_logits(obs_ctx* ctx, const char* who, uint32_t T, uint32_t vocab, int dtype) {
  if (dtype != OBS_LOGITS_F32 && dtype != OBS_LOGITS_BF16)
    return obs::set_error(ctx, OBS_E_INVALID, "%s: dtype must be OBS_LOGITS_F32 or OBS_LOGITS_BF16 (got %d)", who, dtype);
  if (vocab == 0 || vocab > (1u << 24) || T > (1u << 24))
    return obs::set_error(ctx, OBS_E_SHAPE, "%s: vocab must be in [1, 2^24], rows at most 2^24 (got %u, %u)", who, vocab, T);
  return OBS_OK;
}
int check_lm(obs_ctx* ctx, const char* who, uint32_t T, uint32_t in, uint32_t vocab, uint32_t group) {
  if (group != 64u || in == 0 || in % 512u || in > 16384u || vocab == 0 || vocab > (1u << 24) || T > (1u << 24))
    return obs::set_error(ctx, OBS_E_SHAPE,
                          "%s: group must be 64, in a multiple of 512 up to 16,384, vocab in [1, 2^24], rows at most 2^24 (got %u, %u, %u, %u)",
                          who, group, in, vocab, T);
  return OBS_OK;
}

int launch_few(obs_ctx* ctx, const LmArgs& a) {
  const uint32_t grid = std::min(a.tiles, static_cast<uint32_t>(std::max(ctx->num_cus, 1)));
  auto go = [&](auto kernel) {
    OBS_LAUNCH(ctx, "lm_few", kernel<<<grid, 512, 0, ctx->stream>>>(a));
    return int(OBS_OK);
  };
  if (a.T <= 16u) return a.in <= 2048u ? go(lm_few_kernel<1, true>) : go(lm_few_kernel<1, false>);
  return a.in <= 2048u ? go(lm_few_kernel<2, true>) : go(lm_few_kernel<2, false>);
}
template <uint32_t MT>
int launch_many(obs_ctx* ctx, const LmArgs& a, uint8_t* xp, float* xf, uint8_t* xs) {
  const uint32_t ttiles = (a.T + 32u * MT - 1u) / (32u * MT);
  OBS_LAUNCH(ctx, "lm_rows", lm_rows_kernel<MT><<<ttiles * MT * 4u, 512, 0, ctx->stream>>>(a.x, a.T, a.in, xp, xf, xs));
  OBS_LAUNCH(ctx, "lm_many", lm_many_kernel<MT><<<(a.tiles + 7u) / 8u * 8u * ttiles, 256, 0, ctx->stream>>>(a, xp, xf, xs, ttiles));
  return OBS_OK;
}
}  // namespace

extern "C" {

int obs_token_logprobs_workspace(obs_ctx* ctx, uint32_t T, uint32_t vocab, int dtype, uint32_t top_k, size_t* bytes) {
  if (!ctx || !bytes) return OBS_E_INVALID;
  *bytes = 0;
  const char* who = "obs_token_logprobs_workspace";
  int rc = check_logits(ctx, who, T, vocab, dtype);
  if (rc != OBS_OK) return rc;
  const LogitsPlan d = logits_plan(T, vocab, top_k);
  *bytes = d.stat + d.tmax;
  return OBS_OK;
}

int obs_token_logprobs(obs_ctx* ctx, const void* logits, int dtype, uint32_t T, uint32_t vocab, uint32_t ld, const int32_t* tokens,
                       float* logprob, float* entropy, uint32_t top_k, int32_t* top_ids, float* top_logprobs, void* ws,
                       size_t ws_bytes) {
  if (!ctx) return OBS_E_INVALID;
  const char* who = "obs_token_logprobs";
  int rc = check_logits(ctx, who, T, vocab, dtype);
  if (rc == OBS_OK) rc = check_outputs(ctx, who, tokens, logprob, top_k, vocab, top_ids, top_logprobs);
  if (rc != OBS_OK) return rc;
  ld = ld ? ld : vocab;
  if (ld < vocab) return obs::set_error(ctx, OBS_E_SHAPE, "%s: row stride %u holds no row of %u", who, ld, vocab);
  const LogitsPlan d = logits_plan(T, vocab, top_k);
  if (T == 0) return OBS_OK;
  if (!logits || !ws) return obs::set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
  const bool bf16 = dtype == OBS_LOGITS_BF16;
  if (!obs::aligned(logits, bf16 ? 2 : 4) || !obs::aligned(ws, 16))
    return obs::set_error(ctx, OBS_E_ALIGN, "%s: logits must be aligned to their type, the workspace to 16 bytes", who);
  if (ws_bytes < d.stat + d.tmax)
    return obs::set_error(ctx, OBS_E_NOMEM, "%s: workspace %zu bytes < %zu needed", who, ws_bytes, d.stat + d.tmax);
  rc = obs::check_grid(ctx, who, static_cast<uint64_t>(T) * d.parts, 256u);
  if (rc != OBS_OK) return rc;
  obs::DeviceGuard guard(ctx);
  uint8_t* wb = static_cast<uint8_t*>(ws);
  float4* stat = reinterpret_cast<float4*>(wb);
  float* tmax = top_k ? reinterpret_cast<float*>(wb + d.stat) : nullptr;
  const uint8_t* lp = static_cast<const uint8_t*>(logits);
  const size_t row_bytes = static_cast<size_t>(ld) * (bf16 ? 2u : 4u);
  const JoinArgs j{stat, tmax, lp, nullptr, tokens, logprob, entropy, top_ids, top_logprobs, row_bytes, d.parts, d.tiles, 1u, vocab, top_k};
  if (bf16) {
    OBS_LAUNCH(ctx, "logits_part", logits_part_kernel<true><<<T * d.parts, 256, 0, ctx->stream>>>(lp, row_bytes, vocab, d.parts, stat, tmax, d.tiles));
    OBS_LAUNCH(ctx, "logprobs_join", logprobs_join_kernel<true, 0><<<T, 256, 0, ctx->stream>>>(j));
  } else {
    OBS_LAUNCH(ctx, "logits_part", logits_part_kernel<false><<<T * d.parts, 256, 0, ctx->stream>>>(lp, row_bytes, vocab, d.parts, stat, tmax, d.tiles));
    OBS_LAUNCH(ctx, "logprobs_join", logprobs_join_kernel<false, 0><<<T, 256, 0, ctx->stream>>>(j));
  }
  return OBS_OK;
}

int obs_lm_logprobs_workspace(obs_ctx* ctx, uint32_t T, uint32_t in, uint32_t vocab, uint32_t top_k, size_t* bytes) {
  if (!ctx || !bytes) return OBS_E_INVALID;
  *bytes = 0;
  int rc = check_lm(ctx, "obs_lm_logprobs_workspace", T, in, vocab, 64u);
  if (rc != OBS_OK) return rc;
  *bytes = lm_plan(T, in, vocab, top_k).all();
  return OBS_OK;
}

int obs_lm_logprobs(obs_ctx* ctx, const uint16_t* x, const uint32_t* w, const uint16_t* scales, const uint16_t* biases, uint32_t T,
                    uint32_t in, uint32_t vocab, uint32_t group, const int32_t* tokens, float* logprob, float* entropy,
                    uint32_t top_k, int32_t* top_ids, float* top_logprobs, void* ws, size_t ws_bytes) {
  if (!ctx) return OBS_E_INVALID;
  const char* who = "obs_lm_logprobs";
  int rc = check_lm(ctx, who, T, in, vocab, group);
  if (rc == OBS_OK) rc = check_outputs(ctx, who, tokens, logprob, top_k, vocab, top_ids, top_logprobs);
  if (rc != OBS_OK) return rc;
  if (T == 0) return OBS_OK;
  if (!x || !w || !scales || !biases || !ws) return obs::set_error(ctx, OBS_E_INVALID, "%s: null pointer", who);
  if (!obs::aligned(x, 16) || !obs::aligned(w, 16) || !obs::aligned(scales, 16) || !obs::aligned(biases, 16) || !obs::aligned(ws, 16))
    return obs::set_error(ctx, OBS_E_ALIGN, "%s: x, the weight, scales, biases and the workspace must be 16-byte aligned", who);
  const LmPlan d = lm_plan(T, in, vocab, top_k);
  if (ws_bytes < d.all()) return obs::set_error(ctx, OBS_E_NOMEM, "%s: workspace %zu bytes < %zu needed", who, ws_bytes, d.all());
  rc = obs::check_grid(ctx, who, static_cast<uint64_t>(d.tiles + 7u) * ((d.rows + 63u) / 64u), 256u);
  if (rc != OBS_OK) return rc;
  obs::DeviceGuard guard(ctx);
  uint8_t* wb = static_cast<uint8_t*>(ws);
  float4* stat = reinterpret_cast<float4*>(wb);
  float* xt = reinterpret_cast<float*>(wb + d.stat);
  float* logits = top_k ? reinterpret_cast<float*>(wb + d.stat + d.xt) : nullptr;
  uint8_t *xp = wb + d.stat + d.xt + d.logits, *xs = xp + d.xp + d.xf;
  float* xf = reinterpret_cast<float*>(xp + d.xp);
  for (uint32_t t0 = 0; t0 < T; t0 += d.rows) {
    const uint32_t n = std::min(d.rows, T - t0);
    const LmArgs a{x + static_cast<size_t>(t0) * in, w, scales, biases, tokens ? tokens + t0 : nullptr, xt, stat, logits, n, in, vocab, d.tiles, d.ld};
    if (T <= LM_FEW)
      rc = launch_few(ctx, a);
    else
      rc = d.mt == 2u ? launch_many<2>(ctx, a, xp, xf, xs) : launch_many<3>(ctx, a, xp, xf, xs);
    if (rc != OBS_OK) return rc;
    const JoinArgs j{stat, reinterpret_cast<const float*>(stat), reinterpret_cast<const uint8_t*>(logits), xt, a.tokens,
                     logprob ? logprob + t0 : nullptr, entropy ? entropy + t0 : nullptr,
                     top_k ? top_ids + static_cast<size_t>(t0) * top_k : nullptr,
                     top_k ? top_logprobs + static_cast<size_t>(t0) * top_k : nullptr, static_cast<size_t>(d.ld) * sizeof(float),
                     d.tiles, d.tiles, 4u, vocab, top_k};
    if (T <= LM_FEW)
      OBS_LAUNCH(ctx, "logprobs_join", logprobs_join_kernel<false, LM_FEW_COLS><<<n, 256, 0, ctx->stream>>>(j));
    else
      OBS_LAUNCH(ctx, "logprobs_join", logprobs_join_kernel<false, LM_COLS><<<n, 256, 0, ctx->stream>>>(j));
  }
  return OBS_OK;
}

}  // extern "C"
