// obs_paged_prefill.hip — attention of the token rows of a batch of prompts over
// a paged key/value cache (obs_sdpa_paged_prefill), with a sliding window that
// keeps the first tokens visible.
#include "obs_paged.hpp"

namespace {
using namespace obsd;
using obs::most_blocks;
using obs::Paged;
using obs::PagedAttn;
using obs::up256;

// ---------------------------------------------------------------------------
// Token rows of prompts
// ---------------------------------------------------------------------------
// A workgroup takes 384 / G consecutive rows of one sequence and the G heads of
// one kv head: 384 columns, 32 a wave, over the blocks of 32 entries that any of
// them sees (or a part of those, where there are few rows). Keys and values go
// through LDS: a block is 8 + 8 v_mfma_f32_32x32x16_bf16 a wave.
//   S^T [32 entries x 32 columns] = K . Q^T, O^T [dims x 32 columns] += V^T . P: a
// lane (column lane % 32, half lane / 32) keeps its column throughout. Row r of
// the score tile is the block's entry with bits 2 and 3 of r exchanged, so a
// lane's sixteen scores are entries 8 half .. + 7 and 16 + 8 half .. + 7: the
// values of one 16-byte read of a transposed value row, in the order of the
// second product's operand.
// Three waves a SIMD (168 registers) overlap each other's products and softmax.
// Measured against it, at 8,192 rows under a window of 4,096 and at a prompt of
// 5,001: one wave of 64 columns a SIMD 936 and 332 us (a wave issues an
// instruction every four cycles), two of 32 columns with the next block's scores
// beside this one's softmax 602 and 245, this one 581 and 220. More loads in
// flight, LDS reads earlier, two blocks a barrier, wave priorities and the other
// machine schedulers gained nothing.
// The running maximum follows the scores only when they pass it by 2^8 (the sums
// and O are in fp32 and P in bf16, which has fp32's range), so O is hardly ever
// rescaled.
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16_v;

constexpr uint32_t PF_COLS = 384, PF_THREADS = 2u * PF_COLS, PF_TARGET = 256, PF_MIN_CHUNK = 4, PF_WHOLE = 12;
constexpr uint32_t PF_TILES = 1024;  // tiles a kv head at most where they are cut into parts
constexpr float PF_SLACK = 8.0f;

__device__ __forceinline__ Span tile_span(const PagedAttn& p, const RowSpan& r, uint32_t n, uint32_t t0, uint32_t t1) {
  // entry of row t is n - (r1 - t); negative: nothing to see
  const uint32_t hi0 = n + t0 + 1u > r.r1 ? n + t0 + 1u - r.r1 : 0u, hi1 = n + t1 > r.r1 ? n + t1 - r.r1 : 0u;
  return span_of(hi0 ? hi0 - 1u : 0u, hi1, p.window, p.sinks);
}
__device__ __forceinline__ uint32_t row_tiles(const PagedAttn& p, const RowSpan& r) {
  const uint32_t tq = PF_COLS / p.G;
  return (r.r1 - r.r0 + tq - 1u) / tq;
}
__device__ __forceinline__ uint32_t seq_tiles(const Paged& a, const PagedAttn& p, uint32_t b) {
  return b < a.n_seqs ? row_tiles(p, paged_rows(a, b)) : 0u;
}
struct PrefillItem {
  uint32_t b, tile, split, splits, first, place;  // first: the part of the tile's split 0; place: the tile among all
  RowSpan r;  // the sequence's rows
  uint32_t n;  // and entries
};
// Tile `place` of a kv head: sequences in order, in each the last tile (the
// longest) first. b is n_seqs behind the last one.
__device__ __forceinline__ PrefillItem prefill_tile(const Paged& a, const PagedAttn& p, uint32_t place, uint32_t lane) {
  uint32_t acc = 0;
  for (uint32_t base = 0; base < a.n_seqs; base += 64u) {
    RowSpan r{0u, 0u};
    uint32_t n = 0;
    if (base + lane < a.n_seqs) {
      r = paged_rows(a, base + lane);
      n = paged_len(a, base + lane);
    }
    const uint32_t incl = wave_scan_u32(row_tiles(p, r)), all = __builtin_amdgcn_readlane(incl, 63);
    if (place < acc + all) {
      const uint32_t l = uniform(static_cast<uint32_t>(__popcll(__ballot(acc + incl <= place))));
      const uint32_t tile = acc + __builtin_amdgcn_readlane(incl, l) - 1u - place;
      return {base + l, uniform(tile), 0u, 1u, uniform(place), uniform(place),
              {static_cast<uint32_t>(__builtin_amdgcn_readlane(r.r0, l)), static_cast<uint32_t>(__builtin_amdgcn_readlane(r.r1, l))},
              static_cast<uint32_t>(__builtin_amdgcn_readlane(n, l))};
    }
    acc += all;
  }
  return {a.n_seqs, 0u, 0u, 1u, 0u, 0u, {0u, 0u}, 0u};
}
// Part `item` of a kv head where there are few tiles: they are cut into parts of
// nearly one length, a tile's parts together. The waves list all tiles' blocks in
// LDS (s_tile), each wave then plans by the list. (With a sequence's tiles cut
// alike, by its last tile, one prompt of 2,000 took 92.5 us against 68.)
__device__ __forceinline__ PrefillItem prefill_part(const Paged& a, const PagedAttn& p, uint32_t item, uint32_t lane, uint32_t wave,
                                                    uint32_t* s_tile) {
  const uint32_t tq = PF_COLS / p.G;
  auto of = [](uint32_t v, uint32_t l) __attribute__((always_inline)) {
    return static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(static_cast<int>(4u * l), static_cast<int>(v)));
  };
  uint32_t n_tiles = 0;
  for (uint32_t base = 0; base < a.n_seqs; base += 64u) {
    RowSpan r{0u, 0u};
    uint32_t n = 0;
    if (base + lane < a.n_seqs) {
      r = paged_rows(a, base + lane);
      n = paged_len(a, base + lane);
    }
    const uint32_t tiles = row_tiles(p, r), incl = wave_scan_u32(tiles), all = __builtin_amdgcn_readlane(incl, 63);
    for (uint32_t x0 = 64u * wave; x0 < all; x0 += PF_THREADS) {  // uniform per wave
      const uint32_t x = x0 + lane;
      uint32_t l = 0;  // sequences that end at or before tile x
#pragma unroll
      for (uint32_t step = 32; step; step >>= 1) l += of(incl, l + step - 1u) <= x ? step : 0u;
      const RowSpan rl{of(r.r0, l), of(r.r1, l)};
      const uint32_t nl = of(n, l), t0 = rl.r0 + (of(incl, l) - 1u - x) * tq;
      if (x < all && n_tiles + x < PF_TILES) s_tile[n_tiles + x] = tile_span(p, rl, nl, t0, umin(rl.r1, t0 + tq)).nblk;
    }
    n_tiles += all;
  }
  __syncthreads();
  n_tiles = umin(n_tiles, PF_TILES);
  float total = 0.0f, longest = 0.0f;
  for (uint32_t base = 0; base < n_tiles; base += 64u) {
    const float v = base + lane < n_tiles ? static_cast<float>(s_tile[base + lane]) : 0.0f;
    total += wave_sum_asc(v);
    longest = fmaxf(longest, wave_max_f32(v));
  }
  // The shortest parts, in steps of an eighth, of which there are no more than the
  // target (a workgroup fills a CU): the longest one sets the time. The parts of one
  // prompt whose tiles have all lengths begin with the longest tile's, so a second
  // round of its shortest ends early: there no longer than half above the even share.
  const float even = total * static_cast<float>(a.n_kv) / static_cast<float>(p.target);
  uint32_t chunk = 0;
  const uint32_t most = a.n_seqs == 1u && longest * static_cast<float>(n_tiles) > 1.5f * total ? 12u : 16u;
  for (uint32_t k = 8; k <= most; ++k) {
    chunk = max(PF_MIN_CHUNK, static_cast<uint32_t>(__builtin_ceilf(even * static_cast<float>(k) * 0.125f)));
    uint32_t parts = 0;
    for (uint32_t base = 0; base < n_tiles; base += 64u)
      parts += wave_sum_u32(base + lane < n_tiles ? plan_splits(s_tile[base + lane], chunk) : 0u);
    if (parts * a.n_kv <= p.target) break;  // uniform
  }
  uint32_t acc = 0;
  for (uint32_t base = 0; base < n_tiles; base += 64u) {
    const uint32_t splits = base + lane < n_tiles ? plan_splits(s_tile[base + lane], chunk) : 0u;
    const uint32_t incl = wave_scan_u32(splits), all = __builtin_amdgcn_readlane(incl, 63);
    if (item < acc + all) {
      const uint32_t l = static_cast<uint32_t>(__popcll(__ballot(acc + incl <= item)));
      const uint32_t sp = __builtin_amdgcn_readlane(splits, l), first = acc + __builtin_amdgcn_readlane(incl, l) - sp;
      PrefillItem it = prefill_tile(a, p, base + l, lane);
      it.split = uniform(item - first);
      it.splits = uniform(sp);
      it.first = uniform(first);
      return it;
    }
    acc += all;
  }
  return {a.n_seqs, 0u, 0u, 1u, 0u, 0u, {0u, 0u}, 0u};
}

template <uint32_t HD, bool F8>
__global__ void __launch_bounds__(PF_THREADS, 3) paged_prefill_kernel(Paged a, PagedAttn p) {
  constexpr uint32_t KS = HD / 16u, DT = HD / 32u, SZ = F8 ? 1u : 2u;
  constexpr uint32_t KROW = HD + 8u, VROW = 40u;  // padded rows (bf16): no bank is hit twice by eight lanes
  constexpr uint32_t KC = HD * SZ / 16u, VC = 2u * SZ;  // 16-byte chunks of a key row, of a block's value row
  constexpr uint32_t KN = 32u * KC, VN = HD * VC;       // chunks of a block: 512, 256 or 128, at most one a thread
  // Keys and values of two blocks; before and after them a slab a wave, through
  // which queries come in and outputs go out by whole 64-byte runs.
  constexpr uint32_t SLAB = 32u * 80u;  // 32 columns of 64 bytes (+16: bank spread)
  constexpr uint32_t K_BYTES = 2u * 32u * KROW * 2u, V_BYTES = 2u * HD * VROW * 2u, SLABS = PF_THREADS / 64u * SLAB;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[K_BYTES + V_BYTES > SLABS ? K_BYTES + V_BYTES : SLABS];
  uint16_t(*const s_k)[32u * KROW] = reinterpret_cast<uint16_t(*)[32u * KROW]>(s_mem);
  uint16_t(*const s_v)[HD * VROW] = reinterpret_cast<uint16_t(*)[HD * VROW]>(s_mem + K_BYTES);
  __shared__ uint32_t s_bad;  // an edge block holds values that are not finite
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6);
  const uint32_t col = lane & 31u, half = lane >> 5;
  const uint32_t kv = blockIdx.x % a.n_kv;
  __shared__ uint32_t s_tile[PF_TILES];
  const PrefillItem it = p.target ? prefill_part(a, p, blockIdx.x / a.n_kv, lane, wave, s_tile)
                                  : prefill_tile(a, p, blockIdx.x / a.n_kv, lane);
  const uint32_t b = it.b;
  if (b >= a.n_seqs) return;  // uniform
  // everything of the tile in scalar registers: no address or branch below takes the vector unit
  const RowSpan r = it.r;
  const uint32_t n = it.n;
  const uint32_t tq = PF_COLS / p.G, t0r = r.r0 + it.tile * tq, t1r = umin(r.r1, t0r + tq);
  if (tid == 0u && it.tile == 0u && it.split == 0u && kv == 0u && paged_len_bad(a, b)) paged_flag(a.status);
  const Span s = tile_span(p, r, n, t0r, t1r);
  const uint32_t hi_first = n + t0r + 1u > r.r1 ? n + t0r + 1u - r.r1 : 0u;
  const uint32_t lo_last = p.window && s.hi > p.window ? s.hi - p.window : 0u;
  const uint32_t q0 = s.nblk / it.splits, q1 = s.nblk % it.splits;  // parts of q0 or q0 + 1 blocks
  const uint32_t x0 = it.split * q0 + umin(it.split, q1), x1 = x0 + q0 + (it.split < q1 ? 1u : 0u);
  // for the join (row arrays that decrease make more tiles than rows allow: those are dropped)
  if (p.target && it.split == 0u && tid == 0u && it.place * a.n_kv + kv < p.tiles)
    reinterpret_cast<uint4*>(p.plan)[static_cast<size_t>(it.place) * a.n_kv + kv] = make_uint4(it.first, it.splits, t0r, t1r);
  const float scale = F8 ? __uint_as_float(uniform(__float_as_uint(p.scale_log2 * a.k_scale[kv]))) : p.scale_log2;
  if (tid == 0u) s_bad = 0u;

  // the wave's columns: limits, state
  const uint32_t per_g = (65536u + p.G - 1u) / p.G;  // c / G as c * per_g >> 16: exact below 384 columns and up to 16 heads
  auto row_of = [&](uint32_t c) __attribute__((always_inline)) { return c * per_g >> 16; };
  auto is_col = [&](uint32_t c) __attribute__((always_inline)) { return row_of(c) < tq && t0r + row_of(c) < t1r; };
  const uint32_t c = 32u * wave + col, t_row = t0r + row_of(c);
  const bool have = is_col(c);
  const uint32_t hi = have && n + t_row + 1u > r.r1 ? n + t_row + 1u - r.r1 : 0u;
  const uint32_t lo = p.window && hi > p.window ? hi - p.window : 0u;
  // the columns' queries by whole rows (a lane's own column, 16 bytes of a row at a
  // time, would fetch every line four times)
  constexpr uint32_t QC = HD / 8u, QR = 64u / QC;  // 16-byte chunks of a row, rows a load
  u32x4_v qt[HD / 16u];
#pragma unroll
  for (uint32_t i = 0; i < HD / 16u; ++i) {
    const uint32_t qc = 32u * wave + QR * i + lane / QC, qr = row_of(qc);
    const bool ok = is_col(qc);
    qt[i] = *reinterpret_cast<const u32x4_v*>(p.q + static_cast<size_t>(ok ? t0r + qr : 0u) * p.q_ld +
                                              (kv * p.G + (ok ? qc - qr * p.G : 0u)) * HD + 8u * (lane % QC));
    if (!ok) qt[i] = u32x4_v{0u, 0u, 0u, 0u};
  }
  uint8_t* const slab = s_mem + wave * SLAB;
  auto wave_sync = [] __attribute__((always_inline))() {  // a wave's LDS traffic is in order; the compiler keeps it so
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  bf16x8_v qb[KS];
  auto take_queries = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t k4 = 0; k4 < HD / 32u; ++k4) {  // 32 dims at a time
      if (lane % QC / 4u == k4) {
#pragma unroll
        for (uint32_t i = 0; i < HD / 16u; ++i)
          *reinterpret_cast<u32x4_v*>(slab + (QR * i + lane / QC) * 80u + 16u * (lane % 4u)) = qt[i];
      }
      wave_sync();
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j)
        qb[2u * k4 + j] = *reinterpret_cast<const bf16x8_v*>(slab + col * 80u + 32u * j + 16u * half);
      wave_sync();
    }
  };
  float m = NEG_INF, l = 0.0f;
  f32x16_v o[DT];
#pragma unroll
  for (uint32_t d = 0; d < DT; ++d) o[d] = f32x16_v{};

  // A wave's chunks lie in one half of a block, so in one page: a scalar offset
  // and a constant one a lane. The first waves bring keys, others values.
  const uint32_t kc = tid, vc = tid >= 256u ? tid - 256u : tid + 512u;
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
    if (has_k) kr = *reinterpret_cast<const u32x4_v*>(base + koff);
  };
  auto load_v = [&](const Blk& k) __attribute__((always_inline)) {
    const uint8_t* base = a.v + ((static_cast<size_t>(k.iv) * HD << a.lp) + (k.t & pmask)) * SZ;
    if (has_v) vr = *reinterpret_cast<const u32x4_v*>(base + voff);
  };
  auto page_bits = [](const Blk& k) __attribute__((always_inline)) {
    return (k.ok0 ? 0xffffu : 0u) | (k.ok1 ? 0xffff0000u : 0u);
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
    if (has_k) {
      uint16_t* to = &s_k[buf][(kc / KC) * KROW + (16u / SZ) * (kc % KC)];
#pragma unroll
      for (uint32_t j = 0; j < 2u / SZ; ++j) *reinterpret_cast<u32x4_v*>(to + 8u * j) = widen(kr, j);
    }
  };
  // At the edge, values hidden from every row are stored as zero (the pool may
  // hold anything there), and those that are not finite too: the rows that see
  // them get them at the end, and no other row meets them.
  auto store_v = [&](uint32_t buf, const Blk& k) __attribute__((always_inline)) {
    if (has_v) {
      u32x4_v w[2u / SZ];
#pragma unroll
      for (uint32_t j = 0; j < 2u / SZ; ++j) w[j] = widen(vr, j);
      if (k.edge) {  // uniform
        const uint32_t bits = seen_bits(k.t, s.hi, s.lo, p.sinks) & page_bits(k);
        uint32_t bad = 0u;
#pragma unroll
        for (uint32_t j = 0; j < 2u / SZ; ++j) {
          w[j] &= word_masks(bits >> (v_ent + 8u * j));
#pragma unroll
          for (uint32_t q = 0; q < 4; ++q) {
            // all ones in the exponent: adding one in its last place carries into the sign's
            const uint32_t e = (w[j][q] & 0x7f807f80u) + 0x00800080u;
            const uint32_t wild = (e & 0x80008000u) >> 15;  // bit 0, bit 16
            bad |= wild;
            w[j][q] &= ~(wild * 0xffffu);
          }
        }
        if (bad) s_bad = 1u;
      }
#pragma unroll
      for (uint32_t j = 0; j < 2u / SZ; ++j) *reinterpret_cast<u32x4_v*>(&s_v[buf][v_dim * VROW + v_ent + 8u * j]) = w[j];
    }
  };
  auto sees = [&](uint32_t e) __attribute__((always_inline)) { return e < hi && (e >= lo || e < p.sinks); };

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
    Blk ka = block_of(x0), kb = block_of(x0 + 1u);
    load_k(ka);
    load_v(ka);
    take_queries();
    __syncthreads();  // s_bad is zero, the slabs are free
    store_k(x0 & 1u);
    store_v(x0 & 1u, ka);
    __syncthreads();
    for (uint32_t x = x0; x < x1; ++x) {
      if (((x - x0) & 63u) == 62u) fetch_ids(x + 2u);  // uniform
      load_k(kb);  // in flight until the end of the iteration
      load_v(kb);
      __builtin_amdgcn_sched_barrier(0);
      f32x16_v sc;
      scores(x & 1u, sc);
      if (ka.edge) {  // uniform
        auto counts = [&](uint32_t e) { return e < s.hi && (e + 16u > s.lo || e < p.sinks); };
        if (tid == 0u && ((!ka.ok0 && counts(ka.t)) || (!ka.ok1 && counts(ka.t + 16u)))) paged_flag(a.status);
        const uint32_t bits = (seen_bits(ka.t, hi, lo, p.sinks) & page_bits(ka)) >> (8u * half);
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) sc[i] = bits >> (16u * (i / 8u) + i % 8u) & 1u ? sc[i] : NEG_INF;
      }
      maximum(sc);
      const bool up = mx * scale > m + PF_SLACK;
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
#pragma unroll
      for (uint32_t k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (uint32_t d = 0; d < DT; ++d)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              *reinterpret_cast<const bf16x8_v*>(&s_v[x & 1u][(32u * d + col) * VROW + 16u * k2 + 8u * half]), pb[k2], o[d], 0, 0, 0);
      const Blk kn = block_of(x + 2u);
      // the slots of block x - 1, last read before the barrier that began this iteration
      store_k((x + 1u) & 1u);
      store_v((x + 1u) & 1u, kb);
      __syncthreads();
      ka = kb;
      kb = kn;
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
  const float L = l + lane_xor32_f32(l, lane);
  __syncthreads();  // the last block's keys and values were read
  // column and 16-byte chunk that a lane stores of a slab
  const uint32_t ocol = lane / 4u, och = lane % 4u;
  if (it.splits == 1u) {
    const float inv = (F8 ? a.v_scale[kv] : 1.0f) / L;
    uint16_t* to[2];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t oc = 32u * wave + ocol + 16u * j, orow = row_of(oc);
      to[j] = is_col(oc) ? p.out + (static_cast<size_t>(t0r + orow) * p.nh + kv * p.G + oc - orow * p.G) * HD + 8u * och : nullptr;
    }
#pragma unroll
    for (uint32_t d = 0; d < DT; ++d) {
#pragma unroll
      for (uint32_t i = 0; i < 16; i += 4) {
        float v[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) v[j] = L == 0.0f ? 0.0f : o[d][i + j] * inv;
        *reinterpret_cast<uint2*>(slab + col * 80u + 4u * i + 8u * half) =
            make_uint2(pack_bf16_pair_rne(v[0], v[1]), pack_bf16_pair_rne(v[2], v[3]));
      }
      wave_sync();
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j)
        if (to[j])
          *reinterpret_cast<u32x4_v*>(to[j] + 32u * d) = *reinterpret_cast<const u32x4_v*>(slab + (ocol + 16u * j) * 80u + 16u * och);
      wave_sync();
    }
  } else {
    const size_t at = static_cast<size_t>(blockIdx.x) * PF_COLS;
    if (have && half == 0u) {
      p.ml[(at + c) * 2u] = m;
      p.ml[(at + c) * 2u + 1u] = L;
    }
#pragma unroll
    for (uint32_t d = 0; d < 2u * DT; ++d) {  // 16 dims in fp32
#pragma unroll
      for (uint32_t i = 0; i < 8; i += 4) {
        const uint32_t e = 8u * (d & 1u) + i;
        *reinterpret_cast<f32x4_v*>(slab + col * 80u + 8u * i + 16u * half) =
            f32x4_v{o[d / 2u][e], o[d / 2u][e + 1], o[d / 2u][e + 2], o[d / 2u][e + 3]};
      }
      wave_sync();
#pragma unroll
      for (uint32_t j = 0; j < 2; ++j) {
        const uint32_t oc = 32u * wave + ocol + 16u * j;
        if (is_col(oc))
          *reinterpret_cast<u32x4_v*>(p.part + (at + oc) * HD + 16u * d + 4u * och) =
              *reinterpret_cast<const u32x4_v*>(slab + (ocol + 16u * j) * 80u + 16u * och);
      }
      wave_sync();
    }
  }
}

// A tile's parts joined in order: 1024 / HD columns a workgroup, four dims a
// thread, eight parts in flight at once.
template <uint32_t HD, bool F8>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(Paged a, PagedAttn p, uint32_t items) {
  constexpr uint32_t CW = 1024u / HD, WG = PF_COLS / CW;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, place = blockIdx.x / (WG * a.n_kv), kv = blockIdx.x / WG % a.n_kv;
  const uint32_t c = blockIdx.x % WG * CW + tid / (HD / 4u), d = 4u * (tid % (HD / 4u));
  uint32_t tiles = 0;
  for (uint32_t base = 0; base < a.n_seqs; base += 64u)
    tiles += wave_sum_u32(seq_tiles(a, p, base + lane));
  if (place >= tiles) return;  // uniform
  const uint4 plan = reinterpret_cast<const uint4*>(p.plan)[static_cast<size_t>(place) * a.n_kv + kv];
  // (the bounds by items and rows: whatever the row array, nothing outside the buffers is met)
  const uint32_t splits = umin(uniform(plan.y), items), first = umin(uniform(plan.x), items);
  const uint32_t t = plan.z + c / p.G, h = kv * p.G + c % p.G;
  if (splits == 1u || c / p.G >= PF_COLS / p.G || t >= plan.w || t >= a.n_rows) return;
  float M = NEG_INF, L = 0.0f;
  f32x4_v o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t i0 = 0; i0 < splits; i0 += 8u) {
    float2 ml[8];
    f32x4_v x[8];
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      // behind the last part it again, without weight
      const size_t part = umin((first + umin(i0 + i, splits - 1u)) * a.n_kv + kv, items - 1u);
      ml[i] = *reinterpret_cast<const float2*>(p.ml + (part * PF_COLS + c) * 2u);
      x[i] = *reinterpret_cast<const f32x4_v*>(p.part + (part * PF_COLS + c) * HD + d);
    }
    float mn = M;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) mn = fmaxf(mn, ml[i].x);
    const float back = M == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(M - mn);
    M = mn;
    L *= back;
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) o[j] *= back;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      if (i0 + i >= splits) break;  // uniform
      const float f = ml[i].x == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(ml[i].x - mn);
      L = __builtin_fmaf(ml[i].y, f, L);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) o[j] = __builtin_fmaf(x[i][j], f, o[j]);
    }
  }
  const float inv = (F8 ? a.v_scale[kv] : 1.0f) / L;
  float v[4];
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) v[j] = L == 0.0f ? 0.0f : o[j] * inv;
  *reinterpret_cast<uint2*>(p.out + (static_cast<size_t>(t) * p.nh + h) * HD + d) =
      make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

// Prefill: with few rows for the chip (tiles of both kinds of sequence ends
// counted by the rows alone) a tile's blocks are cut into parts, unless the table
// and the window leave a tile at most twelve: up to there the join's launch costs
// more than the parts save (one prompt of 256 19.5 us whole, 23.0 in parts; 384
// 24.2 and 27.5, four of 300 21.2 and 29.2; a row over 400 entries 21.5 and 18.9).
// More tiles than three quarters of the CUs: whole ones end as early (four prompts
// of up to 985 48 us against 54; 2,600 rows of 5,000 entries 201 and 215), but for
// one that the table hardly outgrows, whose tiles have all lengths (2,600 107.7
// whole, 96.6 in parts; 3,000 123.3 and 119.1). All by the table, as the lengths are
// the device's: one of 32,768 entries takes a prompt of 256 from 19.1 to 21.6 us, four
// of 300 from 22.3 to 31.7 and one of 2,600 from 98.5 to 108.2.
struct PrefillPlan {
  uint64_t items, tiles;  // workgroups and tiles (of all kv heads) at most
  bool split;
  size_t ml, part, plan;
  size_t all() const { return ml + part + plan + 256u; }
};
PrefillPlan prefill_plan(const obs_paged_kv* kv, const obs_paged_seqs* s, uint32_t n_heads, uint32_t window, uint32_t sinks) {
  PrefillPlan d{};
  const uint32_t tq = PF_COLS / (n_heads / kv->n_kv);
  const uint64_t full = static_cast<uint64_t>(kv->n_kv) * ((s->n_rows + tq - 1u) / tq);
  // tiles: at most one that is not full a sequence, and none of a sequence without rows
  d.tiles = static_cast<uint64_t>(kv->n_kv) * std::min<uint64_t>(s->n_rows, (s->n_rows + tq - 1u) / tq + s->n_seqs);
  const uint64_t entries = static_cast<uint64_t>(s->max_pages) * kv->page;
  const uint64_t blocks = most_blocks(entries, window ? static_cast<uint64_t>(window) + tq : 0u, sinks);
  const bool steps = s->n_seqs == 1u && !window && 2u * entries < 3u * static_cast<uint64_t>(s->n_rows);
  d.split = full <= (steps ? PF_TARGET : PF_TARGET * 3u / 4u) && d.tiles <= static_cast<uint64_t>(PF_TILES) * kv->n_kv && blocks > PF_WHOLE;
  d.items = d.split ? PF_TARGET + d.tiles + 64u : d.tiles;  // parts of 1 / target of all blocks at least, and one a tile
  if (d.split) {
    d.ml = up256(d.items * PF_COLS * 2u * sizeof(float));
    d.part = up256(d.items * PF_COLS * kv->head_dim * sizeof(float));
    d.plan = up256(d.tiles * sizeof(uint4));
  }
  return d;
}

template <uint32_t HD, bool F8>
int launch_prefill(obs_ctx* ctx, const Paged& a, const PagedAttn& p, const PrefillPlan& d) {
  const uint32_t grid = static_cast<uint32_t>(d.items);
  OBS_LAUNCH(ctx, "paged_prefill", paged_prefill_kernel<HD, F8><<<grid, PF_THREADS, 0, ctx->stream>>>(a, p));
  if (d.split)
    OBS_LAUNCH(ctx, "paged_prefill_join",
               paged_prefill_join_kernel<HD, F8><<<static_cast<uint32_t>(d.tiles) * (PF_COLS * HD / 1024u), 256, 0, ctx->stream>>>(a, p, grid));
  return OBS_OK;
}

}  // namespace

namespace obs {
size_t prefill_paged_ws(const obs_paged_kv* kv, const obs_paged_seqs* s, uint32_t n_heads, uint32_t window, uint32_t sinks) {
  const PrefillPlan d = prefill_plan(kv, s, n_heads, window, sinks);
  return d.all();
}
}  // namespace obs

extern "C" {

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
  rc = obs::check_attn(ctx, who, kv, seqs, nullptr, q, out, n_heads, &q_ld, ws, ws_bytes, d.all());
  if (rc != OBS_OK) return rc;
  if (seqs->n_seqs == 0 || seqs->n_rows == 0) return OBS_OK;
  rc = obs::check_grid(ctx, who, d.items, PF_THREADS);
  if (rc == OBS_OK && d.split) rc = obs::check_grid(ctx, who, d.tiles * (PF_COLS * kv->head_dim / 1024u), 256u);
  if (rc != OBS_OK) return rc;
  obs::DeviceGuard guard(ctx);
  const Paged a = obs::paged_args(ctx, kv, seqs);
  uint8_t* wb = static_cast<uint8_t*>(ws);
  const PagedAttn p{q, out, reinterpret_cast<float*>(wb), reinterpret_cast<float*>(wb + d.ml), nullptr,
                   reinterpret_cast<uint2*>(wb + d.ml + d.part), n_heads, n_heads / kv->n_kv, window, sinks, q_ld, 0u, 0u, d.split ? PF_TARGET : 0u, static_cast<uint32_t>(d.tiles),
                   1.4426950408889634f / __builtin_sqrtf(static_cast<float>(kv->head_dim))};
  const bool f8 = kv->dtype == OBS_KV_E4M3;
  if (kv->head_dim == 128u) return f8 ? launch_prefill<128, true>(ctx, a, p, d) : launch_prefill<128, false>(ctx, a, p, d);
  return f8 ? launch_prefill<64, true>(ctx, a, p, d) : launch_prefill<64, false>(ctx, a, p, d);
}

}  // extern "C"
