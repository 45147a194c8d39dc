// Full-attention layers over a paged KV cache, for a batch of sequences that share a prefix: the
// append of a batch's new rows (per-head norm, RoPE, write to the pages) and the attention with the
// output gate. The arithmetic is that of Attention::forward
// (/root/reference/src/model/qwen3_5.rs:430-474) for every sequence of the batch; the reference
// itself serves one sequence from one contiguous cache (/root/reference/src/model/cache.rs:38-79).
//
// Row (b, t) of a call of T new rows a sequence sits at position len_b - T + t and sees the keys
// [0, position]. A row of negative position (a sequence shorter than T, a padded slot of length 0)
// writes nothing and its output is zero.
#include "kv_pages.h"

namespace {

struct Batch {
  const uint32_t* table;  // [B, stride]
  const int32_t* lens;    // [B]
  int B, stride, max_rows;
};

// rows a sequence holds, whatever the device array says
__device__ __forceinline__ int batch_len(const Batch& b, int seq) { return min(max(b.lens[seq], 0), b.max_rows); }

struct AppendArgs {
  KvLayer l;
  Batch b;
  const bf16_t* qg;    // [B, T, Hq, 2 * hd]
  const bf16_t* kx;    // [B, T, Hkv, hd]
  const bf16_t* vx;
  const bf16_t* qw;    // [hd]
  const bf16_t* kw;
  const float* cos_t;  // [npos, half]
  const float* sin_t;
  bf16_t* q_rot;       // [B, T, Hq, hd]
  int T, Hq, npos, half;
  float eps;
};

// One wavefront a (head, row). The norm and the rotation stay fp32 and are rounded once, on the
// store. (ornith_attn_prep rounds the norm's two products to bf16 as the reference's rms_norm does;
// nothing here is compared bit for bit with a contiguous cache's rows, so the values keep what
// they have.)
template <int PER>
__global__ __launch_bounds__(64) void append_kernel(AppendArgs p) {
  constexpr int HD = 64 * PER;
  const int h = blockIdx.x, row = blockIdx.y, lane = threadIdx.x;
  const int seq = row / p.T, pos = batch_len(p.b, seq) - p.T + (row - seq * p.T);
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.l.Hkv;
  const int hk = is_q ? 0 : is_v ? h - p.Hq - p.l.Hkv : h - p.Hq;
  const bf16_t* src = is_q ? p.qg + ((size_t)row * p.Hq + h) * 2 * HD : (is_v ? p.vx : p.kx) + ((size_t)row * p.l.Hkv + hk) * HD;
  bf16_t* dst;
  bool keep = pos >= 0 && (is_v || pos < p.npos);
  if (is_q) {
    dst = p.q_rot + ((size_t)row * p.Hq + h) * HD;
  } else {
    const uint32_t page = keep ? p.b.table[(size_t)seq * p.b.stride + (pos >> p.l.shift)] : 0;
    keep = keep && page < (uint32_t)p.l.n_pages;  // an id past the pool's end: the row goes nowhere
    dst = (is_v ? p.l.v : p.l.k) + ((((size_t)page * p.l.Hkv + hk) << p.l.shift) + (pos & ((1 << p.l.shift) - 1))) * HD;
  }
  if (!keep) return;
  float x[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = dm_bf2f(src[lane * PER + i]);
  if (!is_v) {
    const bf16_t* w = is_q ? p.qw : p.kw;
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) a = dm_fma(x[i], x[i], a);
    const float inv = dm_rsqrt(dm_wave_sum<64>(a) / (float)HD + p.eps);
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = x[i] * inv * dm_bf2f(w[lane * PER + i]);
    // channel e < half turns with e + half: `half` is a whole number of lanes
    const int hl = p.half / PER;
    const bool low = lane < hl, rot = lane < 2 * hl;
    const size_t e = (size_t)pos * p.half + (low ? lane : lane - hl) * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float other = __shfl(x[i], (low ? lane + hl : lane - hl) & 63, 64);
      if (rot) {
        const float c = p.cos_t[e + i], s = p.sin_t[e + i];
        x[i] = low ? dm_fma(-other, s, x[i] * c) : dm_fma(x[i], c, other * s);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) dst[lane * PER + i] = dm_f2bf(x[i]);
}

struct PagedArgs {
  KvLayer l;
  Batch b;
  const bf16_t* q;   // [B, T, Hq, hd]
  const bf16_t* qg;  // [B, T, Hq, 2 * hd], gate in the second half; null: no gate
  bf16_t* out;       // [B, T, Hq, hd]
  int T, Hq, shared;
  float scale;
};

// One wavefront a (head, row), PER channels a lane, the keys one after another.
template <int PER>
__global__ __launch_bounds__(64) void paged_kernel(PagedArgs p) {
  constexpr int HD = 64 * PER;
  const int h = blockIdx.x, row = blockIdx.y, lane = threadIdx.x;
  const int seq = row / p.T, keys = batch_len(p.b, seq) - p.T + (row - seq * p.T) + 1;
  const int hk = h / (p.Hq / p.l.Hkv);
  const size_t at = ((size_t)row * p.Hq + h) * HD + lane * PER;
  float q[PER], o[PER], m = -DM_INF, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    q[i] = dm_bf2f(p.q[at + i]);
    o[i] = 0.f;
  }
  for (int j = 0; j < keys; ++j) {
    const uint32_t id = p.b.table[(size_t)(j < p.shared ? 0 : seq) * p.b.stride + (j >> p.l.shift)];
    const size_t page = min(id, (uint32_t)p.l.n_pages - 1);
    const size_t r = (((page * p.l.Hkv + hk) << p.l.shift) + (j & ((1 << p.l.shift) - 1))) * HD + lane * PER;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) s = dm_fma(q[i], dm_bf2f(p.l.k[r + i]), s);
    s = dm_wave_sum<64>(s) * p.scale;
    const float mn = s > m ? s : m, ref = mn > -DM_INF ? mn : 0.f;
    const float a = dm_exp(m - ref), w = dm_exp(s - ref);
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = dm_fma(w, dm_bf2f(p.l.v[r + i]), o[i] * a);
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    float y = l == 0.f ? 0.f : o[i] / l;
    if (p.qg) y *= dm_sigmoid_f32(dm_bf2f(p.qg[((size_t)row * p.Hq + h) * 2 * HD + HD + lane * PER + i]));
    p.out[at + i] = dm_f2bf(y);
  }
}

Batch batch_of(const ornith_kv_batch* b) { return Batch{b->d_table, b->d_lens, b->B, b->table_stride, b->max_rows}; }

constexpr int kMaxNewRows = 64;  // new rows a sequence in one call

int rows_check(const ornith_kv_pages* p, const ornith_kv_batch* b, int layer, int T, int Hq, const char* who) {
  if (int rc = kv_pages_check(p, who)) return rc;
  if (int rc = kv_batch_check(p, b, who)) return rc;
  ORN_REQUIRE(layer >= 0 && layer < p->n_layers, "%s: layer %d of %d", who, layer, p->n_layers);
  ORN_REQUIRE(T >= 1 && T <= kMaxNewRows && b->B * T <= 65535, "%s: %d new rows for each of %d sequences (at most %d, 65535 in all)", who, T, b->B,
              kMaxNewRows);
  ORN_REQUIRE(Hq >= p->Hkv && Hq % p->Hkv == 0 && Hq <= 1024, "%s: %d query heads on %d KV heads", who, Hq, p->Hkv);
  return ORNITH_OK;
}

}  // namespace

extern "C" {

int ornith_attn_prep_paged(ornith_ctx* ctx, const ornith_kv_pages* pages, int layer, const ornith_kv_batch* batch, const void* d_qg,
                           const void* d_kx, const void* d_vx, const void* d_q_norm_w, const void* d_k_norm_w, int T, int Hq, int rope_dims,
                           float eps, const float* d_cos, const float* d_sin, int table_npos, void* d_q_rot) {
  if (int rc = rows_check(pages, batch, layer, T, Hq, "attn_prep_paged")) return rc;
  ORN_REQUIRE(d_qg && d_kx && d_vx && d_q_norm_w && d_k_norm_w && d_q_rot, "attn_prep_paged: null argument");
  const int hd = pages->hd, per = hd / 64;
  ORN_REQUIRE(rope_dims >= 0 && rope_dims <= hd && rope_dims % (2 * per) == 0, "attn_prep_paged: %d rotary channels of %d (a multiple of %d)",
              rope_dims, hd, 2 * per);
  ORN_REQUIRE(d_cos && d_sin && table_npos >= batch->max_rows, "attn_prep_paged: no cos / sin tables, or %d positions for %d rows", table_npos,
              batch->max_rows);
  ORN_REQUIRE(ctx, "attn_prep_paged: null context");
  const OrnDevice on(ctx);
  const AppendArgs a{kv_layer(pages, layer), batch_of(batch), (const bf16_t*)d_qg, (const bf16_t*)d_kx, (const bf16_t*)d_vx,
                     (const bf16_t*)d_q_norm_w, (const bf16_t*)d_k_norm_w, d_cos, d_sin, (bf16_t*)d_q_rot, T, Hq, table_npos, rope_dims / 2, eps};
  const dim3 grid(Hq + 2 * pages->Hkv, batch->B * T);
  switch (per) {
    case 1: hipLaunchKernelGGL(append_kernel<1>, grid, dim3(64), 0, ctx->stream, a); break;
    case 2: hipLaunchKernelGGL(append_kernel<2>, grid, dim3(64), 0, ctx->stream, a); break;
    default: hipLaunchKernelGGL(append_kernel<4>, grid, dim3(64), 0, ctx->stream, a); break;
  }
  ORN_LAUNCH_CHECK("append_kernel");
  return ORNITH_OK;
}

int ornith_sdpa_paged_gated(ornith_ctx* ctx, const ornith_kv_pages* pages, int layer, const ornith_kv_batch* batch, const void* d_q_rot,
                            const void* d_qg, int T, int Hq, float scale, void* d_out) {
  if (int rc = rows_check(pages, batch, layer, T, Hq, "sdpa_paged")) return rc;
  ORN_REQUIRE(d_q_rot && d_out, "sdpa_paged: null argument");
  ORN_REQUIRE((((uintptr_t)d_q_rot | (uintptr_t)d_qg | (uintptr_t)d_out) & 15) == 0, "sdpa_paged: operands must be 16-byte aligned");
  ORN_REQUIRE(scale > 0.f && scale < DM_INF, "sdpa_paged: scale %g", scale);
  ORN_REQUIRE(ctx, "sdpa_paged: null context");
  const OrnDevice on(ctx);
  const PagedArgs a{kv_layer(pages, layer), batch_of(batch), (const bf16_t*)d_q_rot, (const bf16_t*)d_qg, (bf16_t*)d_out, T, Hq,
                    batch->shared_rows, scale};
  const dim3 grid(Hq, batch->B * T);
  switch (pages->hd) {
    case 64: hipLaunchKernelGGL(paged_kernel<1>, grid, dim3(64), 0, ctx->stream, a); break;
    case 128: hipLaunchKernelGGL(paged_kernel<2>, grid, dim3(64), 0, ctx->stream, a); break;
    default: hipLaunchKernelGGL(paged_kernel<4>, grid, dim3(64), 0, ctx->stream, a); break;
  }
  ORN_LAUNCH_CHECK("paged_kernel");
  return ORNITH_OK;
}

}  // extern "C"
