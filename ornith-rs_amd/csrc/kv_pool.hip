// The pool of a paged KV cache: which sequence holds which page, who shares it, what is free. All of
// that is host bookkeeping (a few integers a token); the device sees page copies and, when a batch is
// asked for, a launch or two that write its tables. Page ids and lengths reach the device in launch
// arguments, so no call waits for the stream and no host buffer has to outlive one.
// Either launch takes 2.0-2.7 us, for 8 sequences of 104 pages as for 64: a step's extension and descriptor together,
// through the Python binding, 7.3 us for 8 sequences and 13 us for 64.
#include "kv_pages.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {

struct Seq {
  bool open = false;
  int rows = 0;
  std::vector<uint32_t> pages;
  size_t synced = 0;  // leading entries that the device's copy of the table has
};

constexpr int kEdits = 448, kSlots = 448;

struct EditArgs {
  uint32_t at[kEdits], id[kEdits];
};
// entries of the sequences' own tables that changed: table[at[i]] = id[i]
__global__ __launch_bounds__(64) void table_edit_kernel(EditArgs a, uint32_t* table, int n) {
  const int i = blockIdx.x * 64 + threadIdx.x;
  if (i < n) table[a.at[i]] = a.id[i];
}

struct BatchArgs {
  int32_t seq[kSlots], len[kSlots];
};
// the batch's tables from the sequences' own, and their lengths: grid (sequences)
__global__ __launch_bounds__(256) void batch_kernel(BatchArgs a, const uint32_t* table, int max_pages, int words, uint32_t* out, int stride,
                                                    int32_t* lens) {
  const uint32_t* src = table + (size_t)a.seq[blockIdx.x] * max_pages;
  for (int i = threadIdx.x; i < words; i += 256) out[(size_t)blockIdx.x * stride + i] = src[i];
  if (threadIdx.x == 0) lens[blockIdx.x] = a.len[blockIdx.x];
}

}  // namespace

struct ornith_kv_pool {
  ornith_ctx* ctx = nullptr;
  int n_layers = 0, n_pages = 0, page_rows = 0, Hkv = 0, hd = 0, max_seqs = 0, max_pages = 0;
  std::vector<void*> k, v;
  std::vector<int> refs;  // sequences that hold a page; 0: free
  int n_free = 0;
  uint32_t lowest = 0;    // no page below it is free
  std::vector<Seq> seqs;
  uint32_t* d_table = nullptr;  // [max_seqs, max_pages]
  uint32_t* d_batch = nullptr;  // [max_seqs, max_pages]
  int32_t* d_lens = nullptr;    // [max_seqs]

  ornith_kv_pages pages() const { return ornith_kv_pages{n_layers, n_pages, page_rows, Hkv, hd, k.data(), v.data()}; }
  bool has(int s) const { return s >= 0 && s < max_seqs && seqs[s].open; }
  void drop(uint32_t page) {
    if (--refs[page] == 0) {
      ++n_free;
      lowest = std::min(lowest, page);
    }
  }
};

namespace {

#define POOL_TRY(who, ...)                                                                \
  try {                                                                                   \
    __VA_ARGS__                                                                           \
  } catch (const std::bad_alloc&) {                                                       \
    return ornith_fail(ORNITH_ERR_INVALID, "%s: out of host memory", who);                \
  }

// the device copies of the sequences' tables brought up to date
int flush_tables(ornith_kv_pool* p, const int* seqs, int n) {
  EditArgs a;
  int m = 0;
  auto flush = [&]() -> int {
    if (m == 0) return ORNITH_OK;
    hipLaunchKernelGGL(table_edit_kernel, dim3((m + 63) / 64), dim3(64), 0, p->ctx->stream, a, p->d_table, m);
    ORN_LAUNCH_CHECK("table_edit_kernel");
    m = 0;
    return ORNITH_OK;
  };
  for (int i = 0; i < n; ++i) {
    const Seq& s = p->seqs[seqs[i]];
    for (size_t j = s.synced; j < s.pages.size(); ++j) {
      a.at[m] = (uint32_t)((size_t)seqs[i] * p->max_pages + j);
      a.id[m++] = s.pages[j];
      if (m == kEdits)
        if (int rc = flush()) return rc;
    }
  }
  if (int rc = flush()) return rc;
  for (int i = 0; i < n; ++i) p->seqs[seqs[i]].synced = p->seqs[seqs[i]].pages.size();
  return ORNITH_OK;
}

int check_seqs(const ornith_kv_pool* p, const int* seqs, int n, const char* who) {
  ORN_REQUIRE(p, "%s: null pool", who);
  ORN_REQUIRE(n >= 1 && n <= p->max_seqs && seqs, "%s: %d sequences", who, n);
  std::vector<char> seen(p->max_seqs);
  for (int i = 0; i < n; ++i) {
    ORN_REQUIRE(p->has(seqs[i]), "%s: no sequence %d", who, seqs[i]);
    ORN_REQUIRE(!seen[seqs[i]], "%s: sequence %d twice", who, seqs[i]);
    seen[seqs[i]] = 1;
  }
  return ORNITH_OK;
}

}  // namespace

extern "C" {

int ornith_kv_pool_create(ornith_ctx* ctx, int n_layers, int n_pages, int page_rows, int Hkv, int hd, int max_seqs, int max_pages,
                          ornith_kv_pool** out) {
  ORN_REQUIRE(out, "kv_pool_create: out is null");
  ORN_REQUIRE(n_layers >= 1 && n_layers <= 4096, "kv_pool_create: %d layers", n_layers);
  ORN_REQUIRE(max_seqs >= 1 && max_seqs <= 4096 && max_pages >= 1 && max_pages <= n_pages, "kv_pool_create: %d sequences of %d pages (of %d)",
              max_seqs, max_pages, n_pages);
  ORN_REQUIRE((int64_t)max_pages * page_rows <= 1 << 30 && (int64_t)max_seqs * max_pages <= INT32_MAX,
              "kv_pool_create: %d pages of %d rows for %d sequences", max_pages, page_rows, max_seqs);
  POOL_TRY("kv_pool_create", {
    // (the sizes' own checks, with pointers that stand for what is yet to be allocated)
    std::vector<void*> some((size_t)n_layers, reinterpret_cast<void*>(16));
    const ornith_kv_pages shape{n_layers, n_pages, page_rows, Hkv, hd, some.data(), some.data()};
    if (int rc = kv_pages_check(&shape, "kv_pool_create")) return rc;
    ORN_REQUIRE(ctx, "kv_pool_create: null context");
    ornith_kv_pool* p = new ornith_kv_pool();
    *out = p;  // (freed by the way out below if a step fails)
    const int rc = [&]() -> int {
      p->ctx = ctx;
      p->n_layers = n_layers;
      p->n_pages = n_pages;
      p->page_rows = page_rows;
      p->Hkv = Hkv;
      p->hd = hd;
      p->max_seqs = max_seqs;
      p->max_pages = max_pages;
      try {
        p->k.assign(n_layers, nullptr);
        p->v.assign(n_layers, nullptr);
        p->refs.assign(n_pages, 0);
        p->seqs.resize(max_seqs);
        p->n_free = n_pages;
      } catch (const std::bad_alloc&) {
        return ornith_fail(ORNITH_ERR_INVALID, "kv_pool_create: out of host memory");
      }
      const size_t bytes = (size_t)n_pages * Hkv * page_rows * hd * 2;
      for (int i = 0; i < n_layers; ++i) {
        if (int r = ornith_alloc(ctx, bytes, &p->k[i])) return r;
        if (int r = ornith_alloc(ctx, bytes, &p->v[i])) return r;
      }
      const size_t words = (size_t)max_seqs * max_pages * 4;
      if (int r = ornith_alloc(ctx, words, (void**)&p->d_table)) return r;
      if (int r = ornith_alloc(ctx, words, (void**)&p->d_batch)) return r;
      return ornith_alloc(ctx, (size_t)max_seqs * 4, (void**)&p->d_lens);
    }();
    if (rc) {
      ornith_kv_pool_destroy(p);
      *out = nullptr;
    }
    return rc;
  })
}

int ornith_kv_pool_destroy(ornith_kv_pool* p) {
  if (!p) return ORNITH_OK;
  for (void* d : p->k) (void)ornith_free(p->ctx, d);
  for (void* d : p->v) (void)ornith_free(p->ctx, d);
  (void)ornith_free(p->ctx, p->d_table);
  (void)ornith_free(p->ctx, p->d_batch);
  (void)ornith_free(p->ctx, p->d_lens);
  delete p;
  return ORNITH_OK;
}

int ornith_kv_pool_pages(const ornith_kv_pool* p, ornith_kv_pages* out) {
  ORN_REQUIRE(p && out, "kv_pool_pages: null argument");
  *out = p->pages();
  return ORNITH_OK;
}

int ornith_kv_pool_open(ornith_kv_pool* p, int* seq_out) {
  ORN_REQUIRE(p && seq_out, "kv_pool_open: null argument");
  for (int s = 0; s < p->max_seqs; ++s)
    if (!p->seqs[s].open) {
      p->seqs[s].open = true;
      *seq_out = s;
      return ORNITH_OK;
    }
  return ornith_fail(ORNITH_ERR_INVALID, "kv_pool_open: all %d sequences are in use", p->max_seqs);
}

int ornith_kv_pool_fork(ornith_kv_pool* p, int seq, int n, int* seqs_out) {
  ORN_REQUIRE(p && seqs_out && n >= 1, "kv_pool_fork: null argument, or %d forks", n);
  ORN_REQUIRE(p->has(seq), "kv_pool_fork: no sequence %d", seq);
  POOL_TRY("kv_pool_fork", {
    std::vector<int> slots;
    for (int s = 0; s < p->max_seqs && (int)slots.size() < n; ++s)
      if (!p->seqs[s].open) slots.push_back(s);
    ORN_REQUIRE((int)slots.size() == n, "kv_pool_fork: %d of %d sequences are free, %d asked for", (int)slots.size(), p->max_seqs, n);
    const Seq& parent = p->seqs[seq];
    const size_t np = parent.pages.size();
    for (int s : slots) p->seqs[s].pages.reserve(np);
    // nothing below allocates
    for (int i = 0; i < n; ++i) {
      Seq& c = p->seqs[slots[i]];
      c.open = true;
      c.rows = parent.rows;
      c.pages.assign(parent.pages.begin(), parent.pages.end());
      c.synced = 0;
      for (uint32_t id : c.pages) ++p->refs[id];
      seqs_out[i] = slots[i];
    }
    return ORNITH_OK;
  })
}

int ornith_kv_pool_extend(ornith_kv_pool* p, const int* seqs, int n, int rows) {
  POOL_TRY("kv_pool_extend", {
    if (int rc = check_seqs(p, seqs, n, "kv_pool_extend")) return rc;
    ORN_REQUIRE(rows >= 0, "kv_pool_extend: %d rows", rows);
    if (rows == 0) return ORNITH_OK;
    // what is needed: new pages, and copies of shared pages whose free rows will be written (the last
    // holder of one keeps it)
    std::vector<uint32_t> src, dst;
    std::vector<char> copies(n);
    // (a page's holders are counted down as their copies are planned, and up again if the call fails)
    struct Planned {
      ornith_kv_pool* p;
      std::vector<uint32_t>& src;
      bool done = false;
      ~Planned() {
        if (!done)
          for (uint32_t id : src) ++p->refs[id];
      }
    } planned{p, src};
    src.reserve(n);
    size_t need = 0;
    int most = 0;
    for (int i = 0; i < n; ++i) {
      const Seq& s = p->seqs[seqs[i]];
      const int64_t have = (int64_t)s.pages.size(), want = ((int64_t)s.rows + rows + p->page_rows - 1) / p->page_rows;
      ORN_REQUIRE(want <= p->max_pages, "kv_pool_extend: sequence %d would hold %lld pages of at most %d", seqs[i], (long long)want, p->max_pages);
      need += (size_t)(want - have);
      if (s.rows % p->page_rows && p->refs[s.pages.back()] > 1) {
        --p->refs[s.pages.back()];
        copies[i] = 1;
        src.push_back(s.pages.back());
        most = std::max(most, s.rows % p->page_rows);
      }
    }
    need += src.size();
    ORN_REQUIRE(need <= (size_t)p->n_free, "kv_pool_extend: %zu pages needed, %d of %d free", need, p->n_free, p->n_pages);
    for (int i = 0; i < n; ++i) p->seqs[seqs[i]].pages.reserve(((size_t)p->seqs[seqs[i]].rows + rows + p->page_rows - 1) / p->page_rows);
    std::vector<uint32_t> taken;
    for (uint32_t id = p->lowest; taken.size() < need; ++id)
      if (!p->refs[id]) taken.push_back(id);
    dst.assign(taken.begin(), taken.begin() + src.size());
    const ornith_kv_pages pages = p->pages();
    if (!src.empty())
      if (int rc = ornith_kv_pages_copy(p->ctx, &pages, src.data(), dst.data(), (int)src.size(), most)) return rc;
    // nothing below fails
    planned.done = true;
    p->n_free -= (int)need;
    if (need) p->lowest = taken.back() + 1;
    size_t c = 0, t = src.size();
    for (int i = 0; i < n; ++i) {
      Seq& s = p->seqs[seqs[i]];
      if (copies[i]) {
        s.pages.back() = taken[c++];
        p->refs[s.pages.back()] = 1;
        s.synced = std::min(s.synced, s.pages.size() - 1);
      }
      s.rows += rows;
      while ((int64_t)s.pages.size() * p->page_rows < s.rows) {
        p->refs[taken[t]] = 1;
        s.pages.push_back(taken[t++]);
      }
    }
    return ORNITH_OK;
  })
}

int ornith_kv_pool_truncate(ornith_kv_pool* p, int seq, int rows) {
  ORN_REQUIRE(p && p->has(seq), "kv_pool_truncate: no sequence %d", seq);
  Seq& s = p->seqs[seq];
  ORN_REQUIRE(rows >= 0 && rows <= s.rows, "kv_pool_truncate: %d rows of %d", rows, s.rows);
  while (!s.pages.empty() && (int64_t)(s.pages.size() - 1) * p->page_rows >= rows) {
    p->drop(s.pages.back());
    s.pages.pop_back();
  }
  s.synced = std::min(s.synced, s.pages.size());
  s.rows = rows;
  return ORNITH_OK;
}

int ornith_kv_pool_close(ornith_kv_pool* p, int seq) {
  ORN_REQUIRE(p && p->has(seq), "kv_pool_close: no sequence %d", seq);
  if (int rc = ornith_kv_pool_truncate(p, seq, 0)) return rc;
  p->seqs[seq].open = false;
  return ORNITH_OK;
}

int ornith_kv_pool_compact(ornith_kv_pool* p, int* moved) {
  ORN_REQUIRE(p, "kv_pool_compact: null pool");
  POOL_TRY("kv_pool_compact", {
    const uint32_t used = (uint32_t)(p->n_pages - p->n_free);
    std::vector<uint32_t> src, dst, to(p->n_pages);
    uint32_t gap = 0;
    for (uint32_t id = used; id < (uint32_t)p->n_pages; ++id)
      if (p->refs[id]) {
        while (p->refs[gap]) ++gap;  // (as many gaps below `used` as used pages above)
        src.push_back(id);
        dst.push_back(gap++);
      }
    if (!src.empty()) {
      const ornith_kv_pages pages = p->pages();
      if (int rc = ornith_kv_pages_copy(p->ctx, &pages, src.data(), dst.data(), (int)src.size(), p->page_rows)) return rc;
    }
    // nothing below fails
    for (size_t i = 0; i < src.size(); ++i) {
      to[src[i]] = dst[i];
      std::swap(p->refs[dst[i]], p->refs[src[i]]);
    }
    p->lowest = used;
    for (Seq& s : p->seqs)
      for (size_t j = 0; j < s.pages.size(); ++j)
        if (s.pages[j] >= used) {
          s.pages[j] = to[s.pages[j]];
          s.synced = std::min(s.synced, j);
        }
    if (moved) *moved = (int)src.size();
    return ORNITH_OK;
  })
}

int ornith_kv_pool_seq(const ornith_kv_pool* p, int seq, int* rows_out, uint32_t* ids_out, int cap, int* n_ids_out) {
  ORN_REQUIRE(p && p->has(seq), "kv_pool_seq: no sequence %d", seq);
  const Seq& s = p->seqs[seq];
  if (rows_out) *rows_out = s.rows;
  if (n_ids_out) *n_ids_out = (int)s.pages.size();
  if (ids_out) {
    ORN_REQUIRE(cap >= (int)s.pages.size(), "kv_pool_seq: room for %d of %zu page ids", cap, s.pages.size());
    std::copy(s.pages.begin(), s.pages.end(), ids_out);
  }
  return ORNITH_OK;
}

int ornith_kv_pool_stats(const ornith_kv_pool* p, int* pages_used, int* pages_shared, int* seqs_open) {
  ORN_REQUIRE(p, "kv_pool_stats: null pool");
  if (pages_used) *pages_used = p->n_pages - p->n_free;
  if (pages_shared) *pages_shared = (int)std::count_if(p->refs.begin(), p->refs.end(), [](int r) { return r > 1; });
  if (seqs_open) *seqs_open = (int)std::count_if(p->seqs.begin(), p->seqs.end(), [](const Seq& s) { return s.open; });
  return ORNITH_OK;
}

int ornith_kv_pool_load(ornith_kv_pool* p, int seq, int layer, const void* d_k, const void* d_v, int cap, int row0, int rows, int at) {
  ORN_REQUIRE(p && p->has(seq), "kv_pool_load: no sequence %d", seq);
  const Seq& s = p->seqs[seq];
  ORN_REQUIRE(at >= 0 && rows >= 0 && at <= s.rows - rows, "kv_pool_load: rows [%d, +%d) of %d", at, rows, s.rows);
  if (rows == 0) return ORNITH_OK;
  for (int i = at / p->page_rows; i <= (at + rows - 1) / p->page_rows; ++i)
    ORN_REQUIRE(p->refs[s.pages[i]] == 1, "kv_pool_load: page %u is shared", s.pages[i]);
  const ornith_kv_pages pages = p->pages();
  return ornith_kv_pages_load(p->ctx, &pages, layer, d_k, d_v, cap, row0, rows, s.pages.data(), (int)s.pages.size(), at);
}

int ornith_kv_pool_store(ornith_kv_pool* p, int seq, int layer, void* d_k, void* d_v, int cap, int row0, int rows, int at) {
  ORN_REQUIRE(p && p->has(seq), "kv_pool_store: no sequence %d", seq);
  const Seq& s = p->seqs[seq];
  ORN_REQUIRE(at >= 0 && rows >= 0 && at <= s.rows - rows, "kv_pool_store: rows [%d, +%d) of %d", at, rows, s.rows);
  const ornith_kv_pages pages = p->pages();
  return ornith_kv_pages_store(p->ctx, &pages, layer, d_k, d_v, cap, row0, rows, s.pages.data(), (int)s.pages.size(), at);
}

int ornith_kv_pool_batch(ornith_kv_pool* p, const int* seqs, int n, ornith_kv_batch* out) {
  ORN_REQUIRE(out, "kv_pool_batch: out is null");
  POOL_TRY("kv_pool_batch", {
    if (int rc = check_seqs(p, seqs, n, "kv_pool_batch")) return rc;
    const OrnDevice on(p->ctx);
    if (int rc = flush_tables(p, seqs, n)) return rc;
    // the full pages that all of them hold, and the longest
    const Seq& first = p->seqs[seqs[0]];
    int most = 0, least = first.rows;
    size_t words = 0, common = first.pages.size();
    for (int i = 0; i < n; ++i) {
      const Seq& s = p->seqs[seqs[i]];
      most = std::max(most, s.rows);
      least = std::min(least, s.rows);
      words = std::max(words, s.pages.size());
      common = std::min(common, s.pages.size());
      common = (size_t)(std::mismatch(first.pages.begin(), first.pages.begin() + common, s.pages.begin()).first - first.pages.begin());
    }
    for (int i = 0; i < n; i += kSlots) {
      BatchArgs a;
      const int m = std::min(kSlots, n - i);
      for (int j = 0; j < m; ++j) {
        a.seq[j] = seqs[i + j];
        a.len[j] = p->seqs[seqs[i + j]].rows;
      }
      hipLaunchKernelGGL(batch_kernel, dim3(m), dim3(256), 0, p->ctx->stream, a, p->d_table, p->max_pages, (int)words,
                         p->d_batch + (size_t)i * p->max_pages, p->max_pages, p->d_lens + i);
      ORN_LAUNCH_CHECK("batch_kernel");
    }
    *out = ornith_kv_batch{n, p->max_pages, p->d_batch, p->d_lens, (int)std::min(common, (size_t)(least / p->page_rows)) * p->page_rows, most};
    return ORNITH_OK;
  })
}

}  // extern "C"
