// Pages of a KV cache: copies between pages for all layers at once (a fork's last page, a
// compaction), and the way in and out of the contiguous caches that the model's own prompts fill
// (KvCache::update_and_fetch, /root/reference/src/model/cache.rs:38-79; the reference has no pages).
#include "kv_pages.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {

// Ids travel in the launch's arguments: a copy is enqueued without an upload and the caller's
// lists may go away. 4 KB of arguments hold this many.
constexpr int kPairs = 256, kLayers = 64, kIds = 512;

struct CopyArgs {
  bf16_t* pool[2 * kLayers];
  uint32_t src[kPairs], dst[kPairs];
  int runs, run_pieces;  // a page: `runs` stretches (one a KV head, or one for all) of run_pieces 16-byte pieces
  size_t run_stride;     // elements from one stretch to the next
};

// 16 bytes a lane, one piece each: 240 whole pages of 64 rows in ten layers (315 MB read, as much written) take
// 111 us, 5.7 TB/s, the rate of a device copy of which part stays in the cache (one of 2 GiB reaches 4.9).
// Three copies of 29 rows of one page (2.4 MB) take 3.1 us, a launch's worth.
// grid (pieces / 256, pairs, K and V of the layers)
__global__ __launch_bounds__(256) void kv_copy_kernel(CopyArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.runs * a.run_pieces) return;
  const int run = i / a.run_pieces, piece = i - run * a.run_pieces;
  bf16_t* const pool = a.pool[blockIdx.z];
  const size_t page = a.runs * a.run_stride, at = run * a.run_stride + 8 * (size_t)piece;
  const dm_u32x4 v = *reinterpret_cast<const dm_u32x4*>(pool + a.src[blockIdx.y] * page + at);
  *reinterpret_cast<dm_u32x4*>(pool + a.dst[blockIdx.y] * page + at) = v;
}

struct MoveArgs {
  KvLayer l;
  bf16_t* ck;  // [Hkv, cap, hd]
  bf16_t* cv;
  uint32_t ids[kIds];
  int cap, row0, at, rows, row_pieces;  // cache rows [row0, row0 + rows) <-> rows [at, ..) of the pages ids[0], ids[1], ...
};

// 16 bytes a lane: 6621 rows of 2 KV heads of 256 (13.6 MB read, as much written) take 3.7-5 us, 5.4 TB/s and more (out
// of the cache in part), 64 rows 2.4 us, a launch's worth.
// grid (rows x pieces / 256, Hkv, 2)
template <bool LOAD>
__global__ __launch_bounds__(256) void kv_move_kernel(MoveArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x, h = blockIdx.y;
  const int row = i / a.row_pieces, piece = i - row * a.row_pieces, hd = 8 * a.row_pieces;
  if (row >= a.rows) return;
  const int pos = a.at + row;
  const size_t in_page = ((((size_t)a.ids[pos >> a.l.shift] * a.l.Hkv + h) << a.l.shift) + (pos & ((1 << a.l.shift) - 1))) * hd + 8 * piece;
  const size_t in_cache = ((size_t)h * a.cap + a.row0 + row) * hd + 8 * piece;
  dm_u32x4* const p = reinterpret_cast<dm_u32x4*>((blockIdx.z ? a.l.v : a.l.k) + in_page);
  dm_u32x4* const c = reinterpret_cast<dm_u32x4*>((blockIdx.z ? a.cv : a.ck) + in_cache);
  if constexpr (LOAD) *p = *c;
  else *c = *p;
}

// A set of page ids that says whether one was in it already; empty again when it goes.
class Seen {
 public:
  explicit Seen(int n_pages) : bits_(((size_t)n_pages + 63) / 64) {}
  bool has(uint32_t id) const { return bits_[id >> 6] >> (id & 63) & 1; }
  bool add(uint32_t id) {
    const bool was = has(id);
    bits_[id >> 6] |= uint64_t(1) << (id & 63);
    return !was;
  }

 private:
  std::vector<uint64_t> bits_;
};

int move_rows(ornith_ctx* ctx, const ornith_kv_pages* pages, int layer, const void* d_k, const void* d_v, int cap, int row0, int rows,
              const uint32_t* ids, int n_ids, int at, bool load) {
  const char* who = load ? "kv_pages_load" : "kv_pages_store";
  if (int rc = kv_pages_check(pages, who)) return rc;
  ORN_REQUIRE(layer >= 0 && layer < pages->n_layers, "%s: layer %d of %d", who, layer, pages->n_layers);
  ORN_REQUIRE(rows >= 0 && row0 >= 0 && cap >= 0 && row0 <= cap - rows, "%s: rows [%d, +%d) of a cache of %d", who, row0, rows, cap);
  ORN_REQUIRE(n_ids >= 0 && (n_ids == 0 || ids), "%s: %d page ids without their array", who, n_ids);
  const int shift = kv_shift(pages->page_rows);
  ORN_REQUIRE(at >= 0 && (int64_t)at + rows <= std::min<int64_t>((int64_t)n_ids << shift, 1 << 30), "%s: rows [%d, +%d) of %d pages of %d", who, at, rows, n_ids,
              pages->page_rows);
  if (rows == 0) return ORNITH_OK;
  ORN_REQUIRE(d_k && d_v && (((uintptr_t)d_k | (uintptr_t)d_v) & 15) == 0, "%s: null or misaligned cache", who);
  const int first = at >> shift, last = (at + rows - 1) >> shift;
  for (int i = first; i <= last; ++i)
    ORN_REQUIRE(ids[i] < (uint32_t)pages->n_pages, "%s: page %u of %d", who, ids[i], pages->n_pages);
  if (load) {
    try {
      Seen seen(pages->n_pages);
      for (int i = first; i <= last; ++i) ORN_REQUIRE(seen.add(ids[i]), "%s: page %u twice", who, ids[i]);
    } catch (const std::bad_alloc&) {
      return ornith_fail(ORNITH_ERR_INVALID, "%s: out of host memory", who);
    }
  }
  ORN_REQUIRE(ctx, "%s: null context", who);
  const OrnDevice on(ctx);
  MoveArgs a;
  a.l = kv_layer(pages, layer);
  a.ck = (bf16_t*)d_k;
  a.cv = (bf16_t*)d_v;
  a.cap = cap;
  a.row_pieces = pages->hd / 8;
  for (int i = first; i <= last; i += kIds) {
    // the rows on pages ids[i .. i + kIds)
    const int lo = i == first ? at : i << shift, hi = (int)std::min<int64_t>((int64_t)at + rows, (int64_t)(i + kIds) << shift);
    memcpy(a.ids, ids + i, sizeof(uint32_t) * std::min(kIds, last - i + 1));
    a.at = lo - (i << shift);
    a.row0 = row0 + (lo - at);
    a.rows = hi - lo;
    const dim3 grid((unsigned)(((int64_t)a.rows * a.row_pieces + 255) / 256), pages->Hkv, 2);
    if (load) hipLaunchKernelGGL(kv_move_kernel<true>, grid, dim3(256), 0, ctx->stream, a);
    else hipLaunchKernelGGL(kv_move_kernel<false>, grid, dim3(256), 0, ctx->stream, a);
    ORN_LAUNCH_CHECK("kv_move_kernel");
  }
  return ORNITH_OK;
}

}  // namespace

int kv_pages_check(const ornith_kv_pages* p, const char* who) {
  ORN_REQUIRE(p, "%s: null pages", who);
  ORN_REQUIRE(p->n_layers >= 1 && p->d_k && p->d_v, "%s: %d layers, or no pointers to them", who, p->n_layers);
  ORN_REQUIRE(p->n_pages >= 1 && p->Hkv >= 1 && p->Hkv <= 1024, "%s: %d pages of %d KV heads", who, p->n_pages, p->Hkv);
  ORN_REQUIRE(p->page_rows >= 16 && p->page_rows <= 256 && (p->page_rows & (p->page_rows - 1)) == 0,
              "%s: pages of %d rows (a power of two from 16 to 256)", who, p->page_rows);
  ORN_REQUIRE(p->hd == 64 || p->hd == 128 || p->hd == 256, "%s: head width %d (64, 128 or 256)", who, p->hd);
  for (int i = 0; i < p->n_layers; ++i)
    ORN_REQUIRE(p->d_k[i] && p->d_v[i] && (((uintptr_t)p->d_k[i] | (uintptr_t)p->d_v[i]) & 15) == 0,
                "%s: layer %d has null or misaligned pages", who, i);
  return ORNITH_OK;
}

int kv_batch_check(const ornith_kv_pages* p, const ornith_kv_batch* b, const char* who) {
  ORN_REQUIRE(b, "%s: null batch", who);
  ORN_REQUIRE(b->B >= 1 && b->B <= 4096, "%s: %d sequences (1 to 4096)", who, b->B);
  ORN_REQUIRE(b->d_table && b->d_lens && b->table_stride >= 1, "%s: no page tables or lengths", who);
  ORN_REQUIRE(b->max_rows <= 1 << 30, "%s: %d rows a sequence (at most 2^30)", who, b->max_rows);
  ORN_REQUIRE(b->max_rows >= 0 && b->max_rows <= (int64_t)b->table_stride * p->page_rows, "%s: %d rows in %d pages of %d", who, b->max_rows,
              b->table_stride, p->page_rows);
  ORN_REQUIRE(b->shared_rows >= 0 && b->shared_rows % p->page_rows == 0 && b->shared_rows <= b->max_rows,
              "%s: %d shared rows (whole pages of %d, at most %d)", who, b->shared_rows, p->page_rows, b->max_rows);
  return ORNITH_OK;
}

extern "C" {

int ornith_kv_pages_copy(ornith_ctx* ctx, const ornith_kv_pages* pages, const uint32_t* src, const uint32_t* dst, int n, int rows) {
  if (int rc = kv_pages_check(pages, "kv_pages_copy")) return rc;
  ORN_REQUIRE(n >= 0 && (n == 0 || (src && dst)), "kv_pages_copy: %d pairs without their arrays", n);
  ORN_REQUIRE(rows >= 0 && rows <= pages->page_rows, "kv_pages_copy: %d rows of pages of %d", rows, pages->page_rows);
  try {
    Seen written(pages->n_pages);
    for (int i = 0; i < n; ++i) {
      ORN_REQUIRE(src[i] < (uint32_t)pages->n_pages && dst[i] < (uint32_t)pages->n_pages, "kv_pages_copy: page %u to %u of %d", src[i], dst[i],
                  pages->n_pages);
      ORN_REQUIRE(written.add(dst[i]), "kv_pages_copy: page %u is written twice", dst[i]);
    }
    for (int i = 0; i < n; ++i) ORN_REQUIRE(!written.has(src[i]), "kv_pages_copy: page %u is read and written", src[i]);
  } catch (const std::bad_alloc&) {
    return ornith_fail(ORNITH_ERR_INVALID, "kv_pages_copy: out of host memory");
  }
  ORN_REQUIRE(ctx, "kv_pages_copy: null context");
  const OrnDevice on(ctx);
  if (n == 0 || rows == 0) return ORNITH_OK;
  CopyArgs a;
  const bool whole = rows == pages->page_rows;  // the heads' rows lie together
  a.runs = whole ? 1 : pages->Hkv;
  a.run_stride = (size_t)(whole ? pages->Hkv : 1) * pages->page_rows * pages->hd;
  a.run_pieces = (whole ? pages->Hkv : 1) * rows * pages->hd / 8;
  const unsigned gx = (unsigned)((a.runs * a.run_pieces + 255) / 256);
  for (int l = 0; l < pages->n_layers; l += kLayers) {
    const int nl = std::min(kLayers, pages->n_layers - l);
    for (int i = 0; i < nl; ++i) {
      a.pool[2 * i] = static_cast<bf16_t*>(pages->d_k[l + i]);
      a.pool[2 * i + 1] = static_cast<bf16_t*>(pages->d_v[l + i]);
    }
    for (int i = 0; i < n; i += kPairs) {
      const int np = std::min(kPairs, n - i);
      memcpy(a.src, src + i, sizeof(uint32_t) * np);
      memcpy(a.dst, dst + i, sizeof(uint32_t) * np);
      hipLaunchKernelGGL(kv_copy_kernel, dim3(gx, np, 2 * nl), dim3(256), 0, ctx->stream, a);
      ORN_LAUNCH_CHECK("kv_copy_kernel");
    }
  }
  return ORNITH_OK;
}

int ornith_kv_pages_load(ornith_ctx* ctx, const ornith_kv_pages* pages, int layer, const void* d_k_cache, const void* d_v_cache, int cap,
                         int row0, int rows, const uint32_t* ids, int n_ids, int at) {
  return move_rows(ctx, pages, layer, d_k_cache, d_v_cache, cap, row0, rows, ids, n_ids, at, true);
}

int ornith_kv_pages_store(ornith_ctx* ctx, const ornith_kv_pages* pages, int layer, void* d_k_cache, void* d_v_cache, int cap, int row0,
                          int rows, const uint32_t* ids, int n_ids, int at) {
  return move_rows(ctx, pages, layer, d_k_cache, d_v_cache, cap, row0, rows, ids, n_ids, at, false);
}

}  // extern "C"
