// Host side of the paged cache without a GPU: a context that owns no device (for
// the refusals, which come before any device work) and the functions that decide
// what a kernel reads. Built and loaded by test_paged_host.py.
#include "../project-obsidian_amd/csrc/obs_paged.hpp"

extern "C" {
obs_ctx* bare_ctx() {
  obs_ctx* c = new obs_ctx();
  static uint32_t status[obs::CTX_ST_WORDS];
  c->status_dev = status;
  return c;
}
void bare_free(obs_ctx* c) { delete c; }

// span_of: out = {hi, lo, sb, wb, nblk}, then the listed blocks' first entries (at most cap)
void span(uint32_t i0, uint32_t hi, uint32_t window, uint32_t sinks, uint32_t* out, uint32_t cap) {
  const obsd::Span s = obsd::span_of(i0, hi, window, sinks);
  out[0] = s.hi; out[1] = s.lo; out[2] = s.sb; out[3] = s.wb; out[4] = s.nblk;
  for (uint32_t x = 0; x < s.nblk && x < cap; ++x) out[5 + x] = s.start(x);
}
// page id (or -1 where refused), clamped length and rows of one entry
void entry(const int32_t* table, const int32_t* len, const int32_t* row, uint32_t n_pages, uint32_t lp,
           uint32_t n_seqs, uint32_t max_pages, uint32_t n_rows, uint32_t b, uint32_t j, int64_t* out) {
  obs::Paged a{};
  a.table = table; a.len = len; a.row = row;
  a.n_pages = n_pages; a.lp = lp; a.n_seqs = n_seqs; a.max_pages = max_pages; a.n_rows = n_rows;
  bool ok;
  const uint32_t id = obsd::paged_id(a, b, j, ok);
  const obsd::RowSpan r = obsd::paged_rows(a, b);
  out[0] = id; out[1] = ok; out[2] = obsd::paged_len(a, b); out[3] = obsd::paged_len_bad(a, b);
  out[4] = r.r0; out[5] = r.r1;
}
uint32_t rope_rows(uint32_t rope_len) { return obs::rope_rows(rope_len); }
uint32_t seen(uint32_t t, uint32_t hi, uint32_t lo, uint32_t sinks) { return obsd::seen_bits(t, hi, lo, sinks); }
}
