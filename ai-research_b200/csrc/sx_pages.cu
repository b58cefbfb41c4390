// sx_pages.cu -- host bookkeeping of a paged KV cache: free pages, the pages of each sequence.
#include <new>
#include <vector>

#include "sx_host.h"

struct sx_pages {
  uint32_t page_tokens = 0, max_pages = 0;
  std::vector<uint32_t> table;   // [num_seqs][max_pages]
  std::vector<uint32_t> len;     // tokens of each sequence
  std::vector<uint32_t> first;   // pages of it already released from the front
  std::vector<uint32_t> free_;   // last in, first out
};

namespace {

uint32_t pages_of(const sx_pages *p, uint32_t len) {
  return (uint32_t)(((uint64_t)len + p->page_tokens - 1) / p->page_tokens);
}
uint32_t *row_of(sx_pages *p, uint32_t seq) { return p->table.data() + (size_t)seq * p->max_pages; }

sx_status bad(const char *what) {
  sx_host_set_error("%s", what);
  return SX_ERR_INVALID;
}

}  // namespace

extern "C" {

SX_API sx_status sx_pages_create(uint32_t num_pages, uint32_t page_tokens, uint32_t num_seqs,
                                 uint32_t max_pages, sx_pages **out) {
  if (!out || num_pages == 0 || num_pages == SX_NO_PAGE || num_seqs == 0 || max_pages == 0)
    return bad("pages: need out, and pages, sequences and pages per sequence above 0");
  if (page_tokens == 0 || page_tokens % 16 != 0 || page_tokens > 1024)
    return bad("pages: page_tokens must be a multiple of 16, up to 1024");
  if ((uint64_t)max_pages * page_tokens >= (1ull << 31))
    return bad("pages: a sequence must be shorter than 2^31 tokens");
  sx_pages *p = new (std::nothrow) sx_pages();
  if (!p) return SX_ERR_OOM;
  try {
    p->page_tokens = page_tokens;
    p->max_pages = max_pages;
    p->table.assign((size_t)num_seqs * max_pages, SX_NO_PAGE);
    p->len.assign(num_seqs, 0);
    p->first.assign(num_seqs, 0);
    p->free_.resize(num_pages);
    for (uint32_t i = 0; i < num_pages; ++i) p->free_[i] = num_pages - 1 - i;
  } catch (const std::exception &) {
    delete p;
    sx_host_set_error("pages: out of host memory");
    return SX_ERR_OOM;
  }
  *out = p;
  return SX_OK;
}

SX_API void sx_pages_destroy(sx_pages *p) { delete p; }

SX_API sx_status sx_pages_extend(sx_pages *p, uint32_t seq, uint32_t len) {
  if (!p || seq >= p->len.size()) return bad("pages_extend: no such sequence");
  if (len <= p->len[seq]) return SX_OK;
  const uint32_t have = pages_of(p, p->len[seq]), want = pages_of(p, len);
  if (want > p->max_pages) return bad("pages_extend: longer than max_pages pages");
  if (want - have > p->free_.size()) {
    sx_host_set_error("pages_extend: %u pages needed, %zu free", want - have, p->free_.size());
    return SX_ERR_OOM;
  }
  uint32_t *row = row_of(p, seq);
  for (uint32_t i = have; i < want; ++i) {
    row[i] = p->free_.back();
    p->free_.pop_back();
  }
  p->len[seq] = len;
  return SX_OK;
}

SX_API sx_status sx_pages_truncate(sx_pages *p, uint32_t seq, uint32_t len) {
  if (!p || seq >= p->len.size()) return bad("pages_truncate: no such sequence");
  if (len > p->len[seq]) return bad("pages_truncate: longer than the sequence");
  if (len == p->len[seq] && len > 0) return SX_OK;  // (0 ends it, released pages or not)
  uint32_t *row = row_of(p, seq);
  const uint32_t keep = pages_of(p, len);
  if (len > 0 && keep <= p->first[seq])
    return bad("pages_truncate: the last page left has been released");
  for (uint32_t i = pages_of(p, p->len[seq]); i-- > keep;) {
    if (row[i] == SX_NO_PAGE) continue;
    p->free_.push_back(row[i]);  // within the capacity of sx_pages_create
    row[i] = SX_NO_PAGE;
  }
  p->len[seq] = len;
  if (len == 0) p->first[seq] = 0;
  return SX_OK;
}

SX_API sx_status sx_pages_release_before(sx_pages *p, uint32_t seq, uint32_t pos) {
  if (!p || seq >= p->len.size()) return bad("pages_release_before: no such sequence");
  uint32_t *row = row_of(p, seq);
  const uint32_t end = (pos < p->len[seq] ? pos : p->len[seq]) / p->page_tokens;
  for (uint32_t i = p->first[seq]; i < end; ++i) {
    p->free_.push_back(row[i]);
    row[i] = SX_NO_PAGE;
  }
  if (end > p->first[seq]) p->first[seq] = end;
  return SX_OK;
}

SX_API uint32_t sx_pages_length(const sx_pages *p, uint32_t seq) {
  return p && seq < p->len.size() ? p->len[seq] : 0;
}
SX_API uint32_t sx_pages_free_count(const sx_pages *p) {
  return p ? (uint32_t)p->free_.size() : 0;
}
SX_API const uint32_t *sx_pages_table(const sx_pages *p) { return p ? p->table.data() : nullptr; }

}  // extern "C"
