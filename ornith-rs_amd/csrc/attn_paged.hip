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

#include <algorithm>
#include <type_traits>

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

// ---- attention ---------------------------------------------------------------------------------
//
// The keys are cut into a shared part [0, shared), whose rows every query of the batch reads, and a
// part of its own for each sequence; each part into chunks. A workgroup has one chunk, one KV head and
// some 16-row tiles of query rows (a row: one query head of the KV group, one new token, one
// sequence), and leaves (max, sum, values) of its rows over its keys in a slot of the workspace; a
// second launch joins the slots of a row. A call with one chunk in all finishes in the first launch.
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

constexpr int kDies = 8;
constexpr int kChunkPages = 256;  // page ids a workgroup keeps

struct PagedArgs {
  KvLayer l;
  Batch b;
  const bf16_t* q;   // [B, T, Hq, hd]
  const bf16_t* qg;  // [B, T, Hq, 2 * hd], gate in the second half; null: no gate
  bf16_t* out;       // [B, T, Hq, hd]
  float* part_o;     // [slots, B * T * Hq, hd]
  float2* part_ml;   // [slots, B * T * Hq]
  int T, Hq, shared;
  int chunk[2], chunks[2];  // of the shared part and of each own part: keys a chunk, and how many there are
  float c2;                 // scale * log2(e)
};

__device__ __forceinline__ void wg_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// all but the last N of this wavefront's loads have arrived
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | 7 << 4 | 15 << 8);
}

// What a row's result is made of by its last step: o / l, the gate, one rounding.
__device__ __forceinline__ float finish_value(float o, float inv, float gate, bool gated) {
  const float y = o * inv;
  return gated ? y / (1.0f + __builtin_amdgcn_exp2f(-gate * 1.44269504088896341f)) : y;
}

// RW wavefronts of 16 query rows each share a block of BK keys; KW such sets take the chunk's blocks in
// turn and meet at the end.
//
// Both products run transposed, so that a lane owns a query row from the scores to the output and the
// probabilities never leave the registers:
//   S^T[key, row] = K . Q^T    A = 16 keys x 32 channels from LDS, B = the row's channels (registers)
//   O^T[ch, row] += V^T . P^T  A = 16 channels x 32 keys, B = the lane's eight probabilities
// The lane of group g = lane / 16 holds keys 16 n + 4 g + r of its row's scores; an MFMA does not care
// in which order k runs if both operands agree, so the k order of the second product is that of the
// registers: keys 4 g .. + 4 and 16 + 4 g .. + 4 of 32. V^T's eight are two transposing LDS reads of
// four keys each (ds_read_b64_tr_b16), so that K and V both lie in LDS as they do in memory and go there
// without passing a register (buffer loads to LDS; rows past the end read as zeros).
// 32-byte pieces of a row lie permuted by its number, so that eight rows' same piece is on all banks.
template <int HD, int RW, int KW, int BK>
struct Attend {
  static constexpr int NT = 64 * RW * KW, ROWB = HD * 2, TILE = BK * ROWB, NS = HD / 32, NC = HD / 16, NK = BK / 16;
  static constexpr int LPR = HD / 8;            // lanes a row in a load to LDS
  static constexpr int LOADS = TILE / 1024 / RW;  // loads a wavefront makes for a block of keys (or values)
  static constexpr int STAGE = 2 * TILE * KW;
  static constexpr int JOIN = KW > 1 ? KW * RW * 16 * (HD * 4 + 8) : 0;
  static constexpr int LDS = STAGE > JOIN ? STAGE : JOIN;
  static_assert(TILE % (1024 * RW) == 0, "whole loads");

  // which 32-byte slot of its row piece c (of 16 bytes) of row `key` lies in, as a byte offset
  static __device__ __forceinline__ int swz(int key) { return HD >= 128 ? key & 7 : key >> 1 & 3; }
};

template <int HD, int RW, int KW, int BK, bool SHARED>
__global__ __launch_bounds__(64 * RW * KW, KW == 1 ? 2 : 1) void attend_kernel(PagedArgs p) {
  using A = Attend<HD, RW, KW, BK>;
  constexpr int ROWB = A::ROWB, TILE = A::TILE, NS = A::NS, NC = A::NC, NK = A::NK;
  extern __shared__ __align__(1024) unsigned char lds[];
  __shared__ uint32_t ids[kChunkPages];
  const int G = p.Hq / p.l.Hkv, rows = (SHARED ? p.b.B : 1) * p.T * G, tiles = (rows + 16 * RW - 1) / (16 * RW);
  // the tiles of one chunk and KV head go to one die, next to each other: they read the same keys
  const int die = blockIdx.x % kDies, nth = blockIdx.x / kDies, round = nth / tiles, tile = nth - round * tiles;
  int item = round * kDies + die;
  const int chunks = p.chunks[SHARED ? 0 : 1], seqs = SHARED ? 1 : p.b.B;
  if (item >= chunks * seqs * p.l.Hkv) return;
  const int hk = item % p.l.Hkv;
  item /= p.l.Hkv;
  const int chunk = item / seqs, seq = item - chunk * seqs;
  const int k0 = (SHARED ? 0 : p.shared) + chunk * p.chunk[SHARED ? 0 : 1];
  const int k1 = min(k0 + p.chunk[SHARED ? 0 : 1], SHARED ? p.shared : batch_len(p.b, seq));
  const bool finishes = p.chunks[0] + p.chunks[1] == 1;
  if (k0 >= k1 && !finishes) return;  // (no key of the chunk: the join knows)

  const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), set = KW == 1 ? 0 : wave / RW, rw = wave - set * RW;
  // the chunk's page ids
  const int page0 = k0 >> p.l.shift, npages = ((k1 - 1) >> p.l.shift) - page0 + 1;
  for (int i = threadIdx.x; i < npages; i += A::NT)
    ids[i] = min(p.b.table[(size_t)seq * p.b.stride + page0 + i], (uint32_t)p.l.n_pages - 1);

  // this lane's query row
  const int rho = tile * 16 * RW + 16 * rw + l16, rc = (SHARED ? 0 : seq * p.T * G) + min(rho, rows - 1);
  const int r = rc / G, head = hk * G + (rc - r * G), rseq = r / p.T;
  const int vis = batch_len(p.b, rseq) - p.T + (r - rseq * p.T) + 1;  // keys that it sees
  const size_t row_head = (size_t)r * p.Hq + head;
  bf16x8_t qf[NS];
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8_t*>(p.q + row_head * HD + 32 * ks + 8 * lg);
  __syncthreads();

  unsigned char* const kt = lds + set * 2 * TILE;
  unsigned char* const vt = kt + TILE;
  const size_t head_rows = (size_t)1 << p.l.shift;
  // block `blk` of keys or values: piece i of 1 KB holds 1024 / ROWB rows
  auto fetch = [&](const bf16_t* pool, unsigned char* to, int blk) {
    constexpr int RPL = 1024 / ROWB;
#pragma unroll
    for (int i = 0; i < A::LOADS; ++i) {
      const int row0 = (i * RW + rw) * RPL, key = k0 + blk * BK + row0;  // (k0 and blocks are multiples of the rows a load has)
      const bool some = key < k1;
      const uint32_t id = __builtin_amdgcn_readfirstlane(some ? ids[(key >> p.l.shift) - page0] : 0u);
      const int in_page = key & ((1 << p.l.shift) - 1);
      const bf16_t* base = pool + (((size_t)id * p.l.Hkv + hk) * head_rows + (some ? in_page : 0)) * HD;
      const __amdgpu_buffer_rsrc_t buf = dm_buffer(base, some ? min(RPL, k1 - key) * ROWB : 0);
      const int lr = lane / A::LPR, slot = lane % A::LPR;
      const int c = ((slot >> 1) ^ A::swz(row0 + lr)) * 2 + (slot & 1);
      typedef __attribute__((address_space(3))) void lds_t;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_t*)(to + (i * RW + rw) * 1024), 16, lr * ROWB + 16 * c, 0, 0, 0);
    }
  };

  f32x4_t o[NC];
#pragma unroll
  for (int t = 0; t < NC; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_i = -DM_INF, l_i = 0.f;
  const int blocks = (k1 - k0 + BK - 1) / BK, turns = (blocks + KW - 1) / KW;
  fetch(p.l.k, kt, set);
  fetch(p.l.v, vt, set);
  for (int turn = 0; turn < turns; ++turn) {
    const int blk = turn * KW + set, key0 = k0 + blk * BK;
    wait_loads<A::LOADS>();
    wg_barrier();
    f32x4_t st[NK];
#pragma unroll
    for (int n = 0; n < NK; ++n) st[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < NS; ++ks)
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const int key = 16 * n + l16, c = 4 * ks + lg;
        const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(kt + key * ROWB + (((c >> 1) ^ A::swz(key)) << 5) + ((c & 1) << 4));
        st[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[ks], st[n], 0, 0, 0);
      }
    wg_barrier();
    fetch(p.l.k, kt, blk + KW);
    // the online softmax of the lane's row: the reference point of its exponentials moves when the
    // maximum has grown by more than 8 binary orders (probabilities up to 2^8 do no harm, and the
    // final division takes them out)
    float mx = -DM_INF;
    const int lim = min(vis, k1);  // (the shared part may end inside a block)
    const bool masked = __builtin_amdgcn_ballot_w64(key0 + BK > lim) != 0;
    if (masked) {
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key0 + 16 * n + 4 * lg + e >= lim) st[n][e] = -DM_INF;
    }
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, st[n][e]);
    mx = fmaxf(mx, dm_xor_lane<16>(mx));
    mx = fmaxf(mx, dm_xor_lane<32>(mx));
    const bool grow = (mx - m_i) * p.c2 > 8.f;
    const float m_new = grow ? mx : m_i;
    const float alpha = grow ? __builtin_amdgcn_exp2f((m_i - m_new) * p.c2) : 1.f;
    m_i = m_new;
    const float mc = m_new > -DM_INF ? -(m_new * p.c2) : 0.f;
    float rs = 0.f;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        st[n][e] = __builtin_amdgcn_exp2f(dm_fma(st[n][e], p.c2, mc));
        rs += st[n][e];
      }
    l_i = l_i * alpha + rs;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f) != 0) {
#pragma unroll
      for (int t = 0; t < NC; ++t) o[t] *= alpha;
    }
    wait_loads<A::LOADS>();
    wg_barrier();
    // A key that one row of the tile sees and another does not: its probability is 0 there, but 0
    // times a value that is no finite number is none. Blocks with such keys (the last of a sequence)
    // are looked through. If there is one, the product leaves out what is not finite, and that is added
    // key by key to the rows that see it; the other rows keep their bits.
    bool odd = false;
    if (masked && __builtin_amdgcn_ballot_w64(vis > 0 && vis < min(key0 + BK, k1)) != 0) {
      uint32_t bad = 0;
      for (int i = lane; i < TILE / 16; i += 64) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(vt + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= ((w[e] & 0x7f80u) == 0x7f80u) | ((w[e] & 0x7f800000u) == 0x7f800000u);
      }
      odd = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
    }
    bf16x8_t pb[BK / 32];
#pragma unroll
    for (int k2 = 0; k2 < BK / 32; ++k2) {
      u32x4_t w;
      w[0] = dm_f2bf2(st[2 * k2][0], st[2 * k2][1]);
      w[1] = dm_f2bf2(st[2 * k2][2], st[2 * k2][3]);
      w[2] = dm_f2bf2(st[2 * k2 + 1][0], st[2 * k2 + 1][1]);
      w[3] = dm_f2bf2(st[2 * k2 + 1][2], st[2 * k2 + 1][3]);
      pb[k2] = __builtin_bit_cast(bf16x8_t, w);
    }
    auto product = [&](auto only_finite) {
#pragma unroll
      for (int k2 = 0; k2 < BK / 32; ++k2)
#pragma unroll
        for (int t = 0; t < NC; ++t) {
          s16x4_t h[2];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int key = 32 * k2 + 16 * u + 4 * lg + (l16 >> 2);
            typedef __attribute__((address_space(3))) s16x4_t lds4;
            h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vt + key * ROWB + ((t ^ A::swz(key)) << 5) + 8 * (l16 & 3)));
            if constexpr (decltype(only_finite)::value) {
#pragma unroll
              for (int e = 0; e < 4; ++e) h[u][e] = (h[u][e] & 0x7f80) == 0x7f80 ? (short)0 : h[u][e];
            }
          }
          const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
          o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pb[k2], o[t], 0, 0, 0);
        }
    };
    if (!odd) {
      product(std::false_type{});
    } else {
      product(std::true_type{});
#pragma unroll 1
      for (int j = 0; j < BK; ++j) {
        float w = 0.f;
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) w = (j >> 4) == n && (j & 3) == e ? st[n][e] : w;
        w = __shfl(w, l16 + 16 * ((j & 15) >> 2), 64);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
          const u32x2_t v = *reinterpret_cast<const u32x2_t*>(vt + j * ROWB + ((t ^ A::swz(j)) << 5) + 8 * lg);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = e & 1 ? dm_bf2f_hi(v[e >> 1]) : dm_bf2f_lo(v[e >> 1]);
            if (key0 + j < lim && !(__builtin_fabsf(x) < DM_INF)) o[t][e] = dm_fma(w, x, o[t][e]);
          }
        }
      }
    }
    wg_barrier();
    fetch(p.l.v, vt, blk + KW);
  }
  wait_loads<0>();  // (the last turns' requests write zeros: not into the LDS of whoever comes next)
  l_i = l_i + dm_xor_lane<16>(l_i);
  l_i = l_i + dm_xor_lane<32>(l_i);

  int t_lo = 0;  // the first of the channel tiles that this wavefront goes on with
  if constexpr (KW > 1) {
    // the sets' sums meet: every wavefront leaves its own in LDS and takes a share of the channels of all
    static_assert(NC % KW == 0, "whole channel tiles a set");
    wg_barrier();
    f32x4_t* const ob = reinterpret_cast<f32x4_t*>(lds);
    float2* const ml = reinterpret_cast<float2*>(lds + (size_t)KW * RW * 16 * HD * 4);
#pragma unroll
    for (int t = 0; t < NC; ++t) ob[((set * RW + rw) * NC + t) * 64 + lane] = o[t];
    if (lg == 0) ml[(set * RW + rw) * 16 + l16] = make_float2(m_i, l_i);
    __syncthreads();
    float w[KW], m = -DM_INF, l = 0.f;
#pragma unroll
    for (int s = 0; s < KW; ++s) m = fmaxf(m, ml[(s * RW + rw) * 16 + l16].x);
#pragma unroll
    for (int s = 0; s < KW; ++s) {
      const float2 v = ml[(s * RW + rw) * 16 + l16];
      w[s] = v.x > -DM_INF ? __builtin_amdgcn_exp2f((v.x - m) * p.c2) : v.y != v.y ? 1.f : 0.f;
      l += v.y * w[s];
    }
    m_i = m;
    l_i = l;
    t_lo = set * (NC / KW);
#pragma unroll
    for (int u = 0; u < NC / KW; ++u) {
      f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KW; ++s) {
        const f32x4_t v = ob[((s * RW + rw) * NC + t_lo + u) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = dm_fma(v[e], w[s], sum[e]);
      }
      o[u] = sum;
    }
  }
  if (rho >= rows) return;
  const int nt = KW > 1 ? NC / KW : NC;
  if (finishes) {
    const float inv = vis > 0 && l_i != 0.f ? 1.0f / l_i : 0.f;
#pragma unroll
    for (int u = 0; u < nt; ++u) {
      const int ch = 16 * (t_lo + u) + 4 * lg;
      u32x2_t gw = {0, 0};
      if (p.qg) gw = *reinterpret_cast<const u32x2_t*>(p.qg + row_head * 2 * HD + HD + ch);
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = vis > 0 ? finish_value(o[u][e], inv, e & 1 ? dm_bf2f_hi(gw[e >> 1]) : dm_bf2f_lo(gw[e >> 1]), p.qg != nullptr) : 0.f;
      *reinterpret_cast<u32x2_t*>(p.out + row_head * HD + ch) = u32x2_t{dm_f2bf2(y[0], y[1]), dm_f2bf2(y[2], y[3])};
    }
    return;
  }
  const size_t at = (size_t)((SHARED ? 0 : p.chunks[0]) + chunk) * p.b.B * p.T * p.Hq + row_head;
#pragma unroll
  for (int u = 0; u < nt; ++u) *reinterpret_cast<f32x4_t*>(p.part_o + at * HD + 16 * (t_lo + u) + 4 * lg) = o[u];
  if (lg == 0 && t_lo == 0) p.part_ml[at] = make_float2(m_i, l_i);
}

// Joins the slots of a (row, head): four channels a lane. Chunks past what the row sees were not
// computed for it, or hold nothing of it, and are not read.
template <int HD>
__global__ __launch_bounds__(HD / 4) void join_kernel(PagedArgs p) {
  const int r = blockIdx.y, head = blockIdx.x, ch = 4 * threadIdx.x, seq = r / p.T;
  const int vis = batch_len(p.b, seq) - p.T + (r - seq * p.T) + 1;
  const size_t row_head = (size_t)r * p.Hq + head, slot = (size_t)p.b.B * p.T * p.Hq;
  const int ns = vis > 0 ? min(p.chunks[0], (vis + p.chunk[0] - 1) / p.chunk[0]) : 0;
  const int no = vis > p.shared ? min(p.chunks[1], (vis - p.shared + p.chunk[1] - 1) / p.chunk[1]) : 0;
  auto place = [&](int i) { return (size_t)(i < ns ? i : p.chunks[0] + i - ns) * slot + row_head; };
  float m = -DM_INF, l = 0.f;
  for (int i = 0; i < ns + no; ++i) m = fmaxf(m, p.part_ml[place(i)].x);
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < ns + no; ++i) {
    const float2 v = p.part_ml[place(i)];
    const float w = v.x > -DM_INF ? __builtin_amdgcn_exp2f((v.x - m) * p.c2) : v.y != v.y ? 1.f : 0.f;
    l = dm_fma(v.y, w, l);
    if (w != 0.f) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(p.part_o + place(i) * HD + ch);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = dm_fma(x[e], w, o[e]);
    }
  }
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  u32x2_t gw = {0, 0};
  if (p.qg) gw = *reinterpret_cast<const u32x2_t*>(p.qg + row_head * 2 * HD + HD + ch);
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = finish_value(o[e], inv, e & 1 ? dm_bf2f_hi(gw[e >> 1]) : dm_bf2f_lo(gw[e >> 1]), p.qg != nullptr);
  *reinterpret_cast<u32x2_t*>(p.out + row_head * HD + ch) = u32x2_t{dm_f2bf2(y[0], y[1]), dm_f2bf2(y[2], y[3])};
}

template <int HD, int RW, int KW, int BK, bool SHARED>
int launch_part(ornith_ctx* ctx, const PagedArgs& a) {
  using A = Attend<HD, RW, KW, BK>;
  const void* f = reinterpret_cast<const void*>(attend_kernel<HD, RW, KW, BK, SHARED>);
  if (A::LDS > 65536 - 4 * kChunkPages) ORN_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, A::LDS));
  const int64_t rows = (int64_t)(SHARED ? a.b.B : 1) * a.T * (a.Hq / a.l.Hkv), tiles = (rows + 16 * RW - 1) / (16 * RW);
  const int64_t items = (int64_t)a.chunks[SHARED ? 0 : 1] * (SHARED ? 1 : a.b.B) * a.l.Hkv;
  hipLaunchKernelGGL((attend_kernel<HD, RW, KW, BK, SHARED>), dim3((unsigned)((items + kDies - 1) / kDies * kDies * tiles)), dim3(A::NT), A::LDS,
                     ctx->stream, a);
  ORN_LAUNCH_CHECK("attend_kernel");
  return ORNITH_OK;
}

template <int HD>
int attend(ornith_ctx* ctx, PagedArgs a, int max_rows) {
  const int G = a.Hq / a.l.Hkv, own_rows = a.T * G, shared_rows = a.b.B * own_rows;
  // chunks: enough workgroups for every compute unit, no chunk shorter than 256 keys
  auto cut = [&](int part, int keys, int64_t sharers, int rows_a_wg) {
    if (keys <= 0) {
      a.chunk[part] = 1;
      a.chunks[part] = 0;
      return;
    }
    const int64_t wgs = sharers * rows_a_wg;
    const int want = (int)std::max<int64_t>(1, (2 * ctx->compute_units + wgs - 1) / wgs);
    // (whole blocks of 64; a chunk that begins inside a page touches one page more than it has)
    const int most = ((kChunkPages - 1) << a.l.shift) / 64 * 64, len = std::min(std::max(256, ((keys + want - 1) / want + 63) / 64 * 64), most);
    a.chunk[part] = len;
    a.chunks[part] = (keys + len - 1) / len;
  };
  const bool wide_shared = shared_rows > 32, wide_own = own_rows > 32;
  cut(0, a.shared, a.l.Hkv, wide_shared ? (shared_rows + 63) / 64 : (shared_rows + 15) / 16);
  cut(1, max_rows - a.shared, (int64_t)a.l.Hkv * a.b.B, wide_own ? (own_rows + 63) / 64 : (own_rows + 15) / 16);
  const int slots = a.chunks[0] + a.chunks[1];
  const size_t cells = (size_t)a.b.B * a.T * a.Hq;
  if (slots != 1) {
    void* base = nullptr;
    if (int rc = ornith_scratch(ctx, slots * cells * (HD * 4 + 8) + 512, &base)) return rc;
    ScratchCursor sc(base);
    a.part_o = sc.take<float>(slots * cells * HD);
    a.part_ml = sc.take<float2>(slots * cells);
  }
  if (a.chunks[0])
    if (int rc = wide_shared ? launch_part<HD, 4, 1, 64, true>(ctx, a) : launch_part<HD, 1, 4, 32, true>(ctx, a)) return rc;
  if (a.chunks[1])
    if (int rc = wide_own ? launch_part<HD, 4, 1, 64, false>(ctx, a) : launch_part<HD, 1, 4, 32, false>(ctx, a)) return rc;
  if (slots != 1) {
    hipLaunchKernelGGL(join_kernel<HD>, dim3(a.Hq, a.b.B * a.T), dim3(HD / 4), 0, ctx->stream, a);
    ORN_LAUNCH_CHECK("join_kernel");
  }
  return ORNITH_OK;
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
  PagedArgs a{};
  a.l = kv_layer(pages, layer);
  a.b = batch_of(batch);
  a.q = (const bf16_t*)d_q_rot;
  a.qg = (const bf16_t*)d_qg;
  a.out = (bf16_t*)d_out;
  a.T = T;
  a.Hq = Hq;
  a.shared = batch->shared_rows;
  a.c2 = scale * 1.44269504088896341f;
  switch (pages->hd) {
    case 64: return attend<64>(ctx, a, batch->max_rows);
    case 128: return attend<128>(ctx, a, batch->max_rows);
    default: return attend<256>(ctx, a, batch->max_rows);
  }
}

}  // extern "C"
