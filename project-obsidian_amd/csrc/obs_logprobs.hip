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
// load cost 7 of 57 us for 777 rows in bf16). One pass; bound by the reading where rows start at 16
// bytes (777 rows of 151,669 in bf16 52 us, 4.5 TB/s). Other rows are read by single logits (dense, seven of
// eight of them: 167 us).
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

// The largest upper half of a key, its lower 12 bits clear, that at least k of a wave's N x 64 reach.
template <uint32_t N>
__device__ __forceinline__ uint32_t keys_edge(const uint32_t (&keys)[N], uint32_t k) {
  uint32_t e = 0u;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1) {
    uint32_t c = 0;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) c += static_cast<uint32_t>(__popcll(__ballot(keys[i] >= (e | bit))));
    if (c >= k) e |= bit;  // uniform
  }
  return e;
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
  constexpr uint32_t CAP = 1024, SUBS = TILE ? 1u : 4u, PER = TILE ? TILE / 64u : 4u;
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
  float first[8], own = NEG_INF;  // maxima of the first 2,048 tiles, the thread's largest
  // of few lanes' edges the best of four waves is nearly what all threads' is (48 rows of 151,936 logits: k = 20
  // 16 us either way, k = 64 48 and 22)
  const bool wide = k > 32u;
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
    if (wide) {
      s_list[tid] = top_key(own, 0u);
    } else {
      const float e = lanes_edge(own, k);
      if (lane == 0u) s_edge[wave] = e;
    }
  }
  const Stat r = stat_group(a, s_st, lane, wave);  // a barrier: the waves' edges are there, or the threads' maxima
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
  // what k of the 256 threads reach with the maxima that they left in s_list
  auto threads_edge = [&]() __attribute__((always_inline)) {
    uint32_t keys[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) keys[i] = static_cast<uint32_t>(s_list[64u * i + lane] >> 32);
    const uint32_t e = keys_edge<4>(keys, k);
    __syncthreads();
    return e <= static_cast<uint32_t>(NONE_KEY >> 32) ? NEG_INF : key_value(static_cast<uint64_t>(e) << 32);
  };
  const float edge = wide ? threads_edge() : fmaxf(fmaxf(s_edge[0], s_edge[1]), fmaxf(s_edge[2], s_edge[3]));
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
  float low = s_edge[4];
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
  if (low == NEG_INF || p.tiles < 2u * k) {  // uniform: few tiles, some of them short; what k threads reach with all of their logits
    float m = NEG_INF;
    for (uint32_t j = wave; j < rows; j += 4u) {
      float x[PER];
      load(j, x);
#pragma unroll
      for (uint32_t e = 0; e < PER; ++e) m = fmaxf(m, x[e]);
    }
    s_list[tid] = top_key(fmaxf(m, NEG_INF), 0u);
    __syncthreads();
    low = fmaxf(low, threads_edge());
  }
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
  // Of many the k largest by their upper bits, every wave over all (433 rows of 984 logits, k = 15: 13 us,
  // with all of them ranked 90).
  if (n > 128u && n <= CAP) {  // uniform
    constexpr uint32_t PER_LANE = CAP / 64u;
    uint64_t mine[CAP / 256u];
    uint32_t keys[PER_LANE];
#pragma unroll
    for (uint32_t i = 0; i < PER_LANE; ++i) keys[i] = 64u * i + lane < n ? static_cast<uint32_t>(s_list[64u * i + lane] >> 32) : 0u;
#pragma unroll
    for (uint32_t i = 0; i < CAP / 256u; ++i) mine[i] = 256u * i + tid < n ? s_list[256u * i + tid] : 0u;
    const uint32_t e = keys_edge<PER_LANE>(keys, k);
    __syncthreads();
    if (tid == 0u) s_n[1] = 0u;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < CAP / 256u; ++i)
      if (mine[i] && static_cast<uint32_t>(mine[i] >> 32) >= e) list(1u, mine[i]);
    __syncthreads();
    n = uniform(s_n[1]);
  }
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
constexpr uint32_t LM_FEW_COLS = 64;  // vocabulary rows of a workgroup

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
// product with ones. HELD: a wave has one slice, whose rows of x and sums stay in registers. Made for
// 2,048 columns (one token 46 us at 151,936 rows): with 512 or 1,024 six or four of the waves idle (38 and
// 39 us), with 2,560 the second turn has two slices (90).
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
  f32x4_v xsh[HELD ? 4 : 1][NT];  // sums of the groups
  if constexpr (HELD) {
#pragma unroll
    for (uint32_t g = 0; g < 4; ++g)
#pragma unroll
      for (uint32_t m = 0; m < NT; ++m) {
        xsh[g][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xh[g][0][m], ones, zero, 0, 0, 0);
        xsh[g][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xh[g][1][m], ones, xsh[g][m], 0, 0, 0);
      }
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
            if constexpr (HELD)
              xs[m] = xsh[g][m];
            else
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
      // whole waves; of two tiles all eight, which else get out of step (24 tokens 64 us, so 60.5), of one those
      // with tokens (one token 47, else 52)
      if (t < RT && (NT == 2u || t / 4u < (p.T + 3u) / 4u)) {
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

// Many tokens: bound by the matrix units, beside which the weights come apart in the
// vector unit. A nibble masked in place at bits 3:0 (7:4) of a half word is the fp16 number
// q 2^-24 (q 2^-20), subnormal; one packed fma makes s (q - 8) of it, which has at most 8 + 3
// significant bits: exact in fp16, with the scales of a vocabulary row brought to 2^-9 by
// their largest's power of two (below 2^-8 of that they end in fp16's subnormal steps, 2^-15
// of the largest). So a product runs over all columns, and what it leaves out, b + 8 s, meets
// the sums of the groups in products of its own. The rows of x are brought into fp16 by a
// power of two each, the largest to 2^14: exact from 2^-29 of that on, off by 2^-39 of it below.
// (Products of q itself, with the scales as factors of every group's sums, took 1,350 us for
// 2,000 tokens: four vector instructions a product. Those of 8-bit numbers, of which a bf16 x
// has two, drop what lies 2^-13 below the largest of eight products.)
//
// First the rows in the order of the products' operands, [tile of 32 MT rows][group][32
// rows][step][lane] 16 bytes, each row's factor back, and the sums of every group (over
// that factor) in three bf16 parts (24 bits). A wave takes a row.
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
  if (lane == 0u) xf[t] = t < T ? __uint_as_float((ex - 14u) << 23) : 0.0f;
  for (uint32_t c = lane; c < gpad * 8u; c += 64u) {
    const uint32_t g = c / 8u;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (t < T && g < groups) v = *reinterpret_cast<const uint4*>(row + 8u * c);
    const float sum = sum_of_8_lanes(sum8(v));
    if (g < groups) {
      // half c / 4 % 2, step c % 4: columns 0, 4 | 1, 5 | 2, 6 | 3, 7 of the eight
      auto pair = [&](float a, float b) __attribute__((always_inline)) {
        return __builtin_bit_cast(uint32_t, f16x2_of(a * up, b * up));
      };
      *reinterpret_cast<uint4*>(xp + 16u * (((static_cast<size_t>(mt / MT) * groups + g) * MT + mt % MT) * 256u + c % 4u * 64u + 32u * (c / 4u % 2u) + r)) =
          make_uint4(pair(bf16lo(v.x), bf16lo(v.z)), pair(bf16hi(v.x), bf16hi(v.z)), pair(bf16lo(v.y), bf16lo(v.w)),
                     pair(bf16hi(v.y), bf16hi(v.w)));
    }
    if (c % 8u == 0u) {
      float rest = sum * up;
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

// Four waves a workgroup, 32 MT tokens x 32 N vocabulary rows a wave, two or three workgroups a CU:
// the sums at one's end (350 us of 1,335 for 2,000 tokens with one of eight waves) beside the
// other's products. Rows and weights come into LDS past the registers, by whole runs of a row; read
// by the lanes that use them, 32 bytes of 32 rows a load, the weights took 165 us, the scales, two
// bytes each, 150, and the rows through registers and their stores 250. 2,000 tokens take 1,220 to
// 1,300 us by the card, 957 to 1,020 TFLOP/s (a library's bf16 product of 2,048, without the 4 bits:
// 1,214 to 1,220 us, 1,045 to 1,050).
typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
// Global memory to LDS: 16 (4) bytes of every lane from its address to `to` (of the wave) and on.
typedef const __attribute__((address_space(1))) uint32_t* GlobalWords;
typedef __attribute__((address_space(3))) uint32_t* LdsWords;
__device__ __forceinline__ void lds_from16(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<GlobalWords>(reinterpret_cast<uintptr_t>(from)), (LdsWords)to, 16, 0, 0);
}
__device__ __forceinline__ void lds_from4(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<GlobalWords>(reinterpret_cast<uintptr_t>(from)), (LdsWords)to, 4, 0, 0);
}
// A barrier behind a wave's LDS accesses and all its loads but the last N (the fence of
// __syncthreads waits for all).
template <uint32_t N>
__device__ __forceinline__ void barrier_but() {
  static_assert(N < 16u, "the low bits of the counter");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070 | N);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}
template <uint32_t MT, uint32_t N>
struct LmTile {
  static constexpr uint32_t THREADS = 256, ROWS = 32u * MT, COLS = 128u * N, GB = 4u / N;  // GB: groups of a block of weights
  static constexpr uint32_t XB = MT * 4096u, WB = COLS * 32u * GB, SB = COLS * 2u * GB;  // bytes of a group of x, of a block's weights and scales
  static constexpr uint32_t OROW = COLS + 8u, OB = 16u * OROW * 4u, WLDS = WB > OB ? WB : OB;  // 16 rows of logits, at the end in their place
  static constexpr uint32_t HELD = N == 1u && MT <= 2u ? 3u : 2u;                        // workgroups a CU
  static_assert(SB == 4u * THREADS && WB == 64u * THREADS, "five loads a thread");
};
template <uint32_t MT, uint32_t N>
__global__ void __launch_bounds__(256, (LmTile<MT, N>::HELD)) lm_many_kernel(LmArgs p, const uint8_t* __restrict__ xp,
                                                                           const float* __restrict__ xf, const uint8_t* __restrict__ xs,
                                                                           uint32_t ttiles, uint32_t vtiles, uint32_t turn) {
  typedef LmTile<MT, N> L;
  constexpr uint32_t GB = L::GB, RB = 32u * GB, SW = GB / 2u;  // bytes of a row's block, words of its scales
  // (arrays of their own, for the compiler to tell the ones being written from those being read)
  __shared__ __attribute__((aligned(16))) uint8_t s_x0[L::XB], s_x1[L::XB], s_w0[L::WLDS], s_w1[L::WLDS], s_s0[L::SB], s_s1[L::SB];
  __shared__ __attribute__((aligned(16))) int s_back[L::ROWS];  // of a row's factor the exponent, and 118 less
  __shared__ uint32_t s_token[L::ROWS];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wn = uniform(tid >> 6);
  const uint32_t col = lane & 31u, half = lane >> 5;
  // An XCD (blockIdx.x % 8) takes `turn` token tiles, whose rows its L2 holds, through all its column tiles, then the next.
  const uint32_t at = blockIdx.x / 8u, own = (vtiles + 7u) / 8u, t0 = at / (turn * own) * turn, many = umin(turn, ttiles - t0);
  const uint32_t in_turn = at - t0 * own, vt = in_turn / many * 8u + blockIdx.x % 8u, tt = t0 + in_turn % many;
  if (vt >= vtiles) return;  // uniform
  const uint32_t v0 = vt * L::COLS, groups = p.in / 64u, gpad = (groups + 15u) & ~15u, most = p.vocab - 1u - v0;  // last row of the tile
  const uint8_t *wb0 = reinterpret_cast<const uint8_t*>(p.w) + static_cast<size_t>(v0) * (p.in / 2u),
                *sb0 = reinterpret_cast<const uint8_t*>(p.s) + static_cast<size_t>(v0) * (2u * groups),
                *bb0 = reinterpret_cast<const uint8_t*>(p.b) + static_cast<size_t>(v0) * (2u * groups);
  const uint8_t* xg = xp + static_cast<size_t>(tt) * groups * L::XB;
  auto load_x = [&](uint32_t g, uint8_t* to) __attribute__((always_inline)) {
    const uint8_t* base = xg + static_cast<size_t>(umin(g, groups - 1u)) * L::XB;
#pragma unroll
    for (uint32_t i = 0; i < MT; ++i) lds_from16(base + 16u * (tid + 256u * i), to + 16u * (64u * wn + 256u * i));
  };
  // GB groups of every row: 2 GB threads for its weights, SW for the scales. A row's chunks change
  // places by its number, so that the reads below meet every bank once. Behind the last row it again.
  auto load_w = [&](uint32_t block, uint8_t* to, uint8_t* sto) __attribute__((always_inline)) {
    const uint32_t bl = umin(block, groups / GB - 1u);
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t r = (128u / GB) * i + tid / (2u * GB);
      lds_from16(wb0 + RB * bl + (umin(r, most) * (p.in / 2u) + 16u * (tid % (2u * GB) ^ (r >> 1 & (2u * GB - 1u)))), to + 16u * (64u * wn + 256u * i));
    }
    lds_from4(sb0 + 2u * GB * bl + (umin(tid / SW, most) * (2u * groups) + 4u * (tid % SW)), sto + 4u * (64u * wn));
  };
  load_w(0u, s_w0, s_s0);
  load_x(0u, s_x0);
  load_w(1u, s_w1, s_s1);
  if (tid < L::ROWS) {
    const uint32_t t = L::ROWS * tt + tid;
    s_back[tid] = static_cast<int>(__float_as_uint(xf[t]) >> 23) - 245;
    s_token[tid] = p.tokens && t < p.T ? lm_token(p, t) : 0xffffffffu;
  }
  // The largest scale of the lane's vocabulary rows: its exponent (or of the biases 2^90 of it: no
  // sum reaches fp32's range); a half of the wave has every other eight groups.
  const uint32_t steps = gpad / 16u;
  uint32_t cex[N], most_s[N] = {}, most_b[N] = {};
  float down[N];  // brings the scales below 2^-8
  auto params = [&](const uint8_t* from, uint32_t n, uint32_t g) __attribute__((always_inline)) {  // of eight groups from g on
    return *reinterpret_cast<const u32x4_v*>(from + (umin(32u * N * wn + 32u * n + col, most) * (2u * groups) + 2u * umin(g, groups - 8u)));
  };
  for (uint32_t s = 0; s < steps; ++s)
#pragma unroll
    for (uint32_t n = 0; n < N; ++n) {
      const u32x4_v v = params(sb0, n, 16u * s + 8u * half), u = params(bb0, n, 16u * s + 8u * half);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        most_s[n] = max(most_s[n], max(v[i] & 0x7fffu, v[i] >> 16 & 0x7fffu));
        most_b[n] = max(most_b[n], max(u[i] & 0x7fffu, u[i] >> 16 & 0x7fffu));
      }
    }
#pragma unroll
  for (uint32_t n = 0; n < N; ++n) {
    const uint32_t e = max(most_s[n] >> 7, max(most_b[n] >> 7, 90u) - 90u);
    cex[n] = umin(max(e, __float_as_uint(lane_xor32_f32(__uint_as_float(e), lane))), 244u);
    down[n] = __uint_as_float((245u - cex[n]) << 23);
  }
  f32x16_v acc[MT][N];
#pragma unroll
  for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
    for (uint32_t n = 0; n < N; ++n) acc[m][n] = f32x16_v{};
  // the groups' sums with b + 8 s
  for (uint32_t s = 0; s < steps; ++s) {
    const uint32_t g = 16u * s + 8u * half;
    bf16x8_v bb[N][2];
#pragma unroll
    for (uint32_t n = 0; n < N; ++n)
#pragma unroll
      for (uint32_t k = 0; k < 2; ++k) {
        u32x4_v v = params(k ? sb0 : bb0, n, g);
        const float f = k ? 8.0f * down[n] : down[n];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = g < groups ? pack_bf16_pair_rne(bf16lo(v[i]) * f, bf16hi(v[i]) * f) : 0u;
        bb[n][k] = __builtin_bit_cast(bf16x8_v, v);
      }
    bf16x8_v xa[LM_SUMS][MT];
#pragma unroll
    for (uint32_t k = 0; k < LM_SUMS; ++k)
#pragma unroll
      for (uint32_t m = 0; m < MT; ++m)
        xa[k][m] = *reinterpret_cast<const bf16x8_v*>(xs + 16u * (((static_cast<size_t>(tt) * MT + m) * LM_SUMS * steps + k * steps + s) * 64u + lane));
#pragma unroll
    for (uint32_t k = 0; k < LM_SUMS; ++k)
#pragma unroll
      for (uint32_t m = 0; m < MT; ++m)
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
          acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xa[k][m], bb[n][0], acc[m][n], 0, 0, 0);
          acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xa[k][m], bb[n][1], acc[m][n], 0, 0, 0);
        }
  }
  barrier_but<0>();
  load_x(1u, s_x1);
  constexpr uint32_t FR = 4u * MT, RING = MT == 1u ? 2u : 4u;  // fragments of x a group; held at once, fewer than those (the barrier stands between)
  static_assert(RING < FR, "the barrier is before the first of the next group's");
  f16x8_v xa[RING];
  u32x4_v wb[N][4], raw[N];
  uint32_t rs[N], last[N];  // scales; the last word of a group's weights
  f16x2_t mul[N][2], off[N];
  uint32_t roff[N], soff[N];
#pragma unroll
  for (uint32_t n = 0; n < N; ++n) {
    const uint32_t r = 32u * N * wn + 32u * n + col;
    roff[n] = RB * r + 16u * (half ^ (r >> 1 & (2u * GB - 1u)));
    soff[n] = 2u * GB * r;
  }
  auto load_a = [&](const uint8_t* from, uint32_t j) __attribute__((always_inline)) {  // fragment j of a group: step j / MT, rows j % MT
    xa[j % RING] = *reinterpret_cast<const f16x8_v*>(from + 16u * ((j % MT * 4u + j / MT) * 64u + lane));
  };
  auto load_raw = [&](const uint8_t* from, const uint8_t* sfrom, uint32_t place) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t n = 0; n < N; ++n) {
      raw[n] = *reinterpret_cast<const u32x4_v*>(from + (roff[n] ^ 32u * place));
      rs[n] = *reinterpret_cast<const uint16_t*>(sfrom + soff[n] + 2u * place);
    }
  };
  auto scales = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t n = 0; n < N; ++n) {
      const float f = __uint_as_float(rs[n] << 16) * down[n];
      mul[n][0] = f16x2_of(f * 0x1p24f, f * 0x1p24f);
      mul[n][1] = f16x2_of(f * 0x1p20f, f * 0x1p20f);
      off[n] = f16x2_of(-8.0f * f, -8.0f * f);
    }
  };
  // two of the eight weights of word w
  auto apart = [&](uint32_t n, uint32_t s, uint32_t i, uint32_t w) __attribute__((always_inline)) {
    const uint32_t v = (i < 2u ? w : w >> 8) & (i & 1u ? 0x00f000f0u : 0x000f000fu);
    wb[n][s][i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(as_f16x2(v), mul[n][i & 1u], off[n]));
  };
  load_raw(s_w0, s_s0, 0u);
  scales();
#pragma unroll
  for (uint32_t n = 0; n < N; ++n) {
#pragma unroll
    for (uint32_t s = 0; s < 3; ++s)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) apart(n, s, i, raw[n][s]);
    last[n] = raw[n][3];
  }
#pragma unroll
  for (uint32_t j = 0; j < RING; ++j) load_a(s_x0, j);
  // A group is one stream of products without a pause, none of which waits for the one
  // before. Beside them stand the reads of the rows RING fragments ahead and the weights to
  // come: step s makes those of step s - 1 of the next group (step 0 the last ones of its own).
  // The one barrier is where the last of a group's rows and the next one's weights are read,
  // and the next one's rows have come; behind it their places are filled: with the rows of the
  // group after the next, and once a block, when its last group is read, the weights of the
  // block after the next, which have until the second barrier to come.
  auto group = [&](uint32_t g, uint32_t q) __attribute__((always_inline)) {  // q = g % (2 GB)
    uint8_t *const own = q & 1u ? s_x1 : s_x0, *const next = q & 1u ? s_x0 : s_x1;
    const uint32_t wq = (q + 1u) % (2u * GB);
    load_raw(wq / GB ? s_w1 : s_w0, wq / GB ? s_s1 : s_s0, wq % GB);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t s = 0; s < 4; ++s)
#pragma unroll
      for (uint32_t m = 0; m < MT; ++m) {
        const uint32_t j = s * MT + m;
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
          acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xa[j % RING], __builtin_bit_cast(f16x8_v, wb[n][s]), acc[m][n], 0, 0, 0);
          if (n == N - 1u) load_a(j + RING < FR ? own : next, (j + RING) % FR);
#pragma unroll
          for (uint32_t i = m * 4u / MT; i < (m + 1u) * 4u / MT; ++i) apart(n, (s + 3u) % 4u, i, s ? raw[n][s - 1u] : last[n]);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (j == MT - 1u) scales();
        if (j + RING + 1u == FR) {
          if (q % GB == GB - 1u)
            barrier_but<5>();  // the five loads of weights behind the rows
          else
            barrier_but<0>();
          load_x(g + 2u, own);
          __builtin_amdgcn_sched_barrier(0);
          if (q % GB == GB - 2u) load_w((g + GB + 2u) / GB, q / GB ? s_w1 : s_w0, q / GB ? s_s1 : s_s0);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
    for (uint32_t n = 0; n < N; ++n) last[n] = raw[n][3];
  };
  for (uint32_t g = 0; g < groups; g += 2u * GB)  // groups is a multiple of 8
#pragma unroll
    for (uint32_t q = 0; q < 2u * GB; ++q) group(g + q, q);
  barrier_but<0>();
  // 32 rows at a time through LDS, eight threads for a row. (A wave a row, one after another,
  // waited for each row's reductions and token.)
  typedef float(*Rows)[L::OROW];
  const Rows out0 = reinterpret_cast<Rows>(s_w0), out1 = reinterpret_cast<Rows>(s_w1);  // rows 0 to 15, 16 to 31
  const uint32_t part = tid % 8u, orow = tid / 8u;
  const float* mine = orow < 16u ? out0[orow] : out1[orow - 16u];
#pragma unroll
  for (uint32_t m = 0; m < MT; ++m) {
    if (m) __syncthreads();
    int back[16];  // rows and columns of one exponent: neither alone takes a logit out of fp32's range
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) back[i] = s_back[32u * m + 8u * (i / 4u) + 4u * half + i % 4u];
#pragma unroll
    for (uint32_t n = 0; n < N; ++n)
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) (i < 8u ? out0 : out1)[8u * (i / 4u % 2u) + 4u * half + i % 4u][32u * N * wn + 32u * n + col] = __builtin_amdgcn_ldexpf(acc[m][n][i], back[i] + static_cast<int>(cex[n]));
    __syncthreads();
    const uint32_t r = 32u * m + orow, t = L::ROWS * tt + r, k = s_token[r] - v0;
    if (part == 0u && k < L::COLS) p.xt[t] = mine[k];
    float x[16u * N];
#pragma unroll
    for (uint32_t i = 0; i < 4u * N; ++i) {
      const f32x4_v v = *reinterpret_cast<const f32x4_v*>(mine + 32u * i + 4u * part);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e) x[4 * i + e] = v[e];
    }
    lm_sums<L::COLS, 8>(p, x, t, v0, part, t < p.T);
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
  uint32_t rows, mb, nb, tiles, ld;  // token rows of a pass, a workgroup's blocks of 32 rows and of 128 columns
  size_t stat, xt, logits, xp, xf, xs;
  size_t all() const { return stat + xt + logits + xp + xf + xs; }
};
// A workgroup's blocks of 32 rows and of 128 columns, by what a launch takes. `one`: us of 2,048
// columns of x with a workgroup a CU, `all` with as many as CUs hold, both measured; more take
// rounds of those, and a part of one at the end, by the XCD with most columns. (Few columns make
// small workgroups: 70 rows of 3,399 23 us, in tiles of 96 x 256 39. Narrow tiles read weights
// by whole lines: 64 rows of 151,936 78 us, 84 in tiles of 256 columns; many rows want wide ones:
// 2,000 1,220 and 1,358.)
struct LmShape {
  uint32_t m, n, held;
  float one, all;
};
const LmShape& lm_shape(uint32_t rows, uint32_t vocab) {
  static constexpr LmShape shapes[] = {{4, 2, 2, 49.0f, 83.0f}, {3, 2, 2, 40.0f, 69.0f}, {4, 1, 2, 30.0f, 46.0f},
                                       {3, 1, 2, 26.0f, 38.0f}, {2, 1, 3, 23.0f, 45.0f}, {1, 1, 3, 19.0f, 28.0f}};
  const LmShape* best = nullptr;
  float least = 0.0f;
  for (const LmShape& s : shapes) {
    const uint64_t tiles = (vocab + 128u * s.n - 1u) / (128u * s.n), n = ((rows + 31u) / 32u + s.m - 1u) / s.m * ((tiles + 7u) / 8u);
    const float cu = static_cast<float>(n) / 32.0f, held = static_cast<float>(s.held);
    const float us = cu <= 1.0f    ? s.one
                     : cu <= held ? s.one + (s.all - s.one) * (cu - 1.0f) / (held - 1.0f)
                                  : (cu + 0.25f * static_cast<float>(s.n)) / held * s.all;
    if (!best || us < least) best = &s, least = us;
  }
  return *best;
}
LmPlan lm_plan(uint32_t T, uint32_t in, uint32_t vocab, uint32_t k) {
  LmPlan d{};
  // the logits of a pass where alternatives are wanted, and its sums, are of a bounded size
  d.rows = T <= LM_FEW ? T : std::min(T, k ? 256u : 4096u);
  if (T > LM_FEW) {
    const LmShape& shape = lm_shape(d.rows, vocab);
    d.mb = shape.m;
    d.nb = shape.n;
  }
  const uint32_t cols = T <= LM_FEW ? LM_FEW_COLS : 128u * d.nb;
  d.tiles = (vocab + cols - 1u) / cols;
  d.ld = (vocab + 3u) & ~3u;
  const size_t groups = in / 64u, gpad = (groups + 15u) & ~size_t(15), blocks = T > LM_FEW ? (d.rows + 32u * d.mb - 1u) / (32u * d.mb) * d.mb : 0u;
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
template <uint32_t MT, uint32_t N>
int launch_many(obs_ctx* ctx, const LmArgs& a, uint8_t* xp, float* xf, uint8_t* xs) {
  typedef LmTile<MT, N> L;
  const uint32_t ttiles = (a.T + L::ROWS - 1u) / L::ROWS, vtiles = (a.vocab + L::COLS - 1u) / L::COLS;
  const uint32_t turn = std::max(1u, (5u << 19) / (a.in / 64u * L::XB));  // 2.5 MB of an XCD's 4 MB of L2
  OBS_LAUNCH(ctx, "lm_rows", lm_rows_kernel<MT><<<ttiles * MT * 4u, 512, 0, ctx->stream>>>(a.x, a.T, a.in, xp, xf, xs));
  OBS_LAUNCH(ctx, "lm_many", lm_many_kernel<MT, N><<<(vtiles + 7u) / 8u * 8u * ttiles, L::THREADS, 0, ctx->stream>>>(
                                 a, xp, xf, xs, ttiles, vtiles, turn));
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
  rc = obs::check_grid(ctx, who, static_cast<uint64_t>(d.tiles + 7u) * ((d.rows + 63u) / 64u), 512u);
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
      rc = d.nb == 1u ? (d.mb == 1u   ? launch_many<1, 1>(ctx, a, xp, xf, xs)
                         : d.mb == 2u ? launch_many<2, 1>(ctx, a, xp, xf, xs)
                         : d.mb == 3u ? launch_many<3, 1>(ctx, a, xp, xf, xs)
                                      : launch_many<4, 1>(ctx, a, xp, xf, xs))
                      : (d.mb == 3u ? launch_many<3, 2>(ctx, a, xp, xf, xs) : launch_many<4, 2>(ctx, a, xp, xf, xs));
    if (rc != OBS_OK) return rc;
    const JoinArgs j{stat, reinterpret_cast<const float*>(stat), reinterpret_cast<const uint8_t*>(logits), xt, a.tokens,
                     logprob ? logprob + t0 : nullptr, entropy ? entropy + t0 : nullptr,
                     top_k ? top_ids + static_cast<size_t>(t0) * top_k : nullptr,
                     top_k ? top_logprobs + static_cast<size_t>(t0) * top_k : nullptr, static_cast<size_t>(d.ld) * sizeof(float),
                     d.tiles, d.tiles, 4u, vocab, top_k};
    if (T <= LM_FEW)
      OBS_LAUNCH(ctx, "logprobs_join", logprobs_join_kernel<false, LM_FEW_COLS><<<n, 256, 0, ctx->stream>>>(j));
    else if (d.nb == 1u)
      OBS_LAUNCH(ctx, "logprobs_join", logprobs_join_kernel<false, 128><<<n, 256, 0, ctx->stream>>>(j));
    else
      OBS_LAUNCH(ctx, "logprobs_join", logprobs_join_kernel<false, 256><<<n, 256, 0, ctx->stream>>>(j));
  }
  return OBS_OK;
}

}  // extern "C"
