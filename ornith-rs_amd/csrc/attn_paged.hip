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

// One wavefront a (head, row): inv = rsqrt(mean x^2 + eps), x inv w, and channel e turned against e + half by
// the position's angle. A chain of latencies (length, page, row; norm across the lanes), with no work to
// speak of: 3.2 us at 8 rows of 20 heads of 256 (160 KB), 4.5 us at 256 rows (5.2 MB; a copy of it takes
// 1.1 us), where one launch after another takes 3.9-4.9 us either way, by the machine. The row itself and the
// norm's weights do not wait for the page: that took 0.6 us off.
// The norm and the rotation stay fp32 and are rounded once, on the store. (ornith_attn_prep rounds the
// norm's two products to bf16 as the reference's rms_norm does; nothing here is compared bit for bit with
// a contiguous cache's rows, so the values keep what they have.)
template <int PER>
__global__ __launch_bounds__(64) void append_kernel(AppendArgs p) {
  constexpr int HD = 64 * PER;
  const int h = blockIdx.x, row = blockIdx.y, lane = threadIdx.x;
  const int seq = row / p.T, pos = batch_len(p.b, seq) - p.T + (row - seq * p.T);
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.l.Hkv;
  const int hk = is_q ? 0 : is_v ? h - p.Hq - p.l.Hkv : h - p.Hq;
  const bf16_t* src = is_q ? p.qg + ((size_t)row * p.Hq + h) * 2 * HD : (is_v ? p.vx : p.kx) + ((size_t)row * p.l.Hkv + hk) * HD;
  float x[PER], w[PER];  // (asked for before the page is looked up)
#pragma unroll
  for (int i = 0; i < PER; ++i) x[i] = dm_bf2f(src[lane * PER + i]);
  if (!is_v) {
#pragma unroll
    for (int i = 0; i < PER; ++i) w[i] = dm_bf2f((is_q ? p.qw : p.kw)[lane * PER + i]);
  }
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
  if (!is_v) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) a = dm_fma(x[i], x[i], a);
    const float inv = dm_rsqrt(dm_wave_sum<64>(a) / (float)HD + p.eps);
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = x[i] * inv * w[i];
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

// What this wavefront (or, with a barrier, the workgroup) has read of LDS is in registers: it may be written again.
template <bool SHARED_BLOCK>
__device__ __forceinline__ void reads_done() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);
  if (SHARED_BLOCK) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// The results of matrix instructions may be read eight wait states after the last of them (16 x 16 x 32). Where
// the reader is in another block that two paths lead to, the compiler counts along one of them only and
// leaves the shorter one without its wait: a row's maximum was then now and then taken from a partial
// sum, which moved the reference point of its exponentials and with it the last bits of the result.
template <int N>
__device__ __forceinline__ void settle(f32x4_t (&v)[N]) {
  static_assert(N == 1 || N == 4, "of a block's scores");
  if constexpr (N == 1) asm volatile("s_nop 7" : "+v"(v[0]));
  else asm volatile("s_nop 7" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
}
// All but the last N of this wavefront's (the workgroup's wavefronts') loads have arrived.
template <int N, bool SHARED_BLOCK>
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | 7 << 4 | 15 << 8);
  if (SHARED_BLOCK) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The least value among a wavefront's rows, one in each of N neighbouring lanes, the same in all groups of N.
template <int N>
__device__ __forceinline__ int least_of_rows(int v) {
#pragma unroll
  for (int s = N / 2; s; s >>= 1) v = min(v, __shfl_xor(v, s, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// The last step of four channels of a row: values / sum, the gate, one rounding. Zeros for a row that sees no key, whatever
// its gate; one whose scores are all minus infinity has the sum 0, and no number comes out.
template <int HD>
__device__ __forceinline__ void store_result(const PagedArgs& p, size_t row_head, int ch, const f32x4_t& o, float l, bool sees) {
  const float inv = 1.0f / l;
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = o[e] * inv;
  if (p.qg) {
    const u32x2_t gw = *reinterpret_cast<const u32x2_t*>(p.qg + row_head * 2 * HD + HD + ch);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float g = e & 1 ? dm_bf2f_hi(gw[e >> 1]) : dm_bf2f_lo(gw[e >> 1]);
      y[e] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g * 1.44269504088896341f));
    }
  }
  *reinterpret_cast<u32x2_t*>(p.out + row_head * HD + ch) = sees ? u32x2_t{dm_f2bf2(y[0], y[1]), dm_f2bf2(y[2], y[3])} : u32x2_t{0, 0};
}

// A workgroup of four wavefronts works in one of two forms:
//   RW = 4, BK = 64  four wavefronts of 16 query rows share a block of 64 keys
//   RW = 1, BK = 16  16 query rows; every wavefront has a block of 16 keys of its own in turn, and their
//                    sums meet at the end (few rows: what counts is how much is in flight)
// Both take 64 KB of LDS at a head width of 256 (the second one 512 bytes more, where its sums meet), two
// workgroups a compute unit.
//
// Both products run transposed, so that a lane owns a query row from the scores to the output and the
// probabilities never leave the registers:
//   S^T[key, row] = K . Q^T    A = 16 keys x 32 channels from LDS, B = the row's channels (registers)
//   O^T[ch, row] += V^T . P^T  A = 16 channels x 32 (16) keys, B = the lane's eight (four) probabilities
// The lane of group g = lane / 16 holds keys 16 n + 4 g + r of its row's scores; an MFMA does not care
// in which order k runs if both operands agree, so the k order of the second product is that of the
// registers: keys 4 g .. + 4 and 16 + 4 g .. + 4 of 32. V^T's eight are two transposing LDS reads of
// four keys each (ds_read_b64_tr_b16), so that K and V both lie in LDS as they do in memory and go there
// without passing a register (buffer loads to LDS; rows past the end read as zeros).
// 32-byte pieces of a row lie permuted by its number, so that eight rows' same piece is on all banks.
constexpr int kWaves = 4;

template <int HD, int RW, int BK>
struct Attend {
  static constexpr int KW = kWaves / RW, ROWB = HD * 2, TILE = BK * ROWB, NS = HD / 32, NC = HD / 16, NK = BK / 16;
  static constexpr int LPR = HD / 8, RPL = 64 / LPR;  // lanes a row, rows a load to LDS
  static constexpr int GROUPS = BK / 16 / RW;         // of 16 rows, which lie on one page, that a wavefront fetches of a block
  static constexpr int PER_GROUP = 16 / RPL, LOADS = GROUPS * PER_GROUP;
  static constexpr int STAGE = 2 * TILE * KW;
  static constexpr int JOIN = KW > 1 ? kWaves * 16 * (HD * 4 + 8) : 0;
  static constexpr int LDS = STAGE > JOIN ? STAGE : JOIN;
  static_assert(BK % (16 * RW) == 0 && (BK == 16 || BK % 32 == 0), "whole groups");

  // which 32-byte slot of a row its first one lies in
  static __device__ __forceinline__ int swz(int row) { return HD >= 128 ? row & 7 : row >> 1 & 3; }
};

template <int HD, int RW, int BK, bool SHARED>
__device__ __forceinline__ void attend_part(const PagedArgs& p, int block, unsigned char* lds, uint32_t* ids) {
  using A = Attend<HD, RW, BK>;
  constexpr int ROWB = A::ROWB, TILE = A::TILE, NS = A::NS, NC = A::NC, NK = A::NK, KW = A::KW;
  const int G = p.Hq / p.l.Hkv, rows = (SHARED ? p.b.B : 1) * p.T * G, tiles = (rows + 16 * RW - 1) / (16 * RW);
  // the tiles of one chunk and KV head go to one die, next to each other: they read the same keys
  const int die = block % kDies, nth = block / kDies, round = nth / tiles, tile = nth - round * tiles;
  int item = round * kDies + die;
  const int chunk_len = p.chunk[SHARED ? 0 : 1], chunks = p.chunks[SHARED ? 0 : 1], seqs = SHARED ? 1 : p.b.B;
  if (item >= chunks * seqs * p.l.Hkv) return;
  const int hk = item % p.l.Hkv;
  item /= p.l.Hkv;
  const int chunk = item / seqs, seq = item - chunk * seqs;
  const int k0 = (SHARED ? 0 : p.shared) + chunk * chunk_len;
  const int k1 = min(k0 + chunk_len, SHARED ? p.shared : batch_len(p.b, seq));
  const bool finishes = p.chunks[0] + p.chunks[1] == 1;
  if (k0 >= k1 && !finishes) return;  // (no key of the chunk: the join knows)

  const int lane = threadIdx.x & 63, l16 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), set = KW == 1 ? 0 : wave, rw = KW == 1 ? wave : 0;
  // the chunk's page ids
  const int page0 = k0 >> p.l.shift, npages = ((k1 - 1) >> p.l.shift) - page0 + 1;
  for (int i = threadIdx.x; i < npages; i += 64 * kWaves)
    ids[i] = min(p.b.table[(size_t)seq * p.b.stride + page0 + i], (uint32_t)p.l.n_pages - 1);

  // this lane's query row
  const int rho = tile * 16 * RW + 16 * rw + l16, rc = (SHARED ? 0 : seq * p.T * G) + min(rho, rows - 1);
  const int r = rc / G, head = hk * G + (rc - r * G), rseq = r / p.T;
  const int vis = batch_len(p.b, rseq) - p.T + (r - rseq * p.T) + 1;  // keys that it sees
  const int least_vis = least_of_rows<16>(vis);
  const size_t row_head = (size_t)r * p.Hq + head;
  bf16x8_t qf[NS];
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8_t*>(p.q + row_head * HD + 32 * ks + 8 * lg);
  __syncthreads();

  // The byte of a group's memory that the lane takes in load i: row i RPL + lane / LPR, the piece that its slot
  // in LDS holds. The numbers' bits lie apart, so load i's is load 0's with a constant's bits turned.
  const int lr = lane / A::LPR, slot = lane % A::LPR;
  const uint32_t at0 = lr * ROWB + 32 * ((slot >> 1) ^ A::swz(lr)) + 16 * (slot & 1);
  // the page of 16-row group g of this wavefront's part of a block (any id where there is no key)
  auto page_of = [&](int blk, int g) {
    const int key = k0 + blk * BK + 16 * (g * RW + rw);
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)ids[min((key >> p.l.shift) - page0, kChunkPages - 1)]);
  };
  auto fetch = [&](const bf16_t* pool, unsigned char* to, int blk, const uint32_t (&page)[A::GROUPS]) {
#pragma unroll
    for (int g = 0; g < A::GROUPS; ++g) {
      const int key = k0 + blk * BK + 16 * (g * RW + rw), have = min(16, k1 - key);
      const size_t first = ((((size_t)page[g] * p.l.Hkv + hk) << p.l.shift) + (key & ((1 << p.l.shift) - 1))) * HD;
      const __amdgpu_buffer_rsrc_t buf = dm_buffer(pool + (have > 0 ? first : 0), have > 0 ? have * ROWB : 0);
#pragma unroll
      for (int i = 0; i < A::PER_GROUP; ++i) {
        typedef __attribute__((address_space(3))) void lds_t;
        const uint32_t turned = (uint32_t)(i * A::RPL * ROWB + 32 * A::swz(i * A::RPL));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (lds_t*)(to + (g * RW + rw) * 16 * ROWB + i * 1024), 16, at0 ^ turned, 0, 0, 0);
      }
    }
  };
  static_assert(ROWB * A::RPL == 1024 && (HD < 128 || A::RPL <= 4), "a load is 1 KB of rows; its first row's number ends in zeros");

  f32x4_t o[NC];
#pragma unroll
  for (int t = 0; t < NC; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m_i = -DM_INF, l_i = 0.f;
  const int blocks = (k1 - k0 + BK - 1) / BK, turns = (blocks + KW - 1) / KW;
  // turns whose blocks every row of the wavefronts sees in full: no masks, and no values to look through
  const int whole = max(0, min(least_vis, k1) - k0) / (BK * KW);
  uint32_t page[A::GROUPS];
#pragma unroll
  for (int g = 0; g < A::GROUPS; ++g) page[g] = page_of(set, g);
  // (The two tiles come as parameters that are told apart: behind a request into LDS the compiler has every
  // read of LDS that may be of the same bytes wait for all requests in flight.)
  auto walk = [&](unsigned char* __restrict__ kt, unsigned char* __restrict__ vt) __attribute__((always_inline)) {
  fetch(p.l.k, kt, set, page);
  fetch(p.l.v, vt, set, page);
  auto one_block = [&](int turn, auto edge) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge)::value;
    const int blk = turn * KW + set, key0 = k0 + blk * BK;
#pragma unroll
    for (int g = 0; g < A::GROUPS; ++g) page[g] = page_of(blk + KW, g);
    wait_loads<A::LOADS, KW == 1>();
    // ---- S^T = K Q^T, the fragments of a step leaving LDS under the products of the step before
    f32x4_t st[NK];
#pragma unroll
    for (int n = 0; n < NK; ++n) st[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    {
      constexpr int STEP = NS < 4 / NK ? NS : 4 / NK, FR = STEP * NK;  // channels' steps at a time: four fragments
      bf16x8_t kf[2][FR];
      auto read = [&](int s, bf16x8_t (&f)[FR]) {
#pragma unroll
        for (int u = 0; u < FR; ++u) {
          const int key = 16 * (u % NK) + l16, c = 4 * (s * STEP + u / NK) + lg;
          f[u] = *reinterpret_cast<const bf16x8_t*>(kt + key * ROWB + (((c >> 1) ^ A::swz(key)) << 5) + ((c & 1) << 4));
        }
      };
      static_assert(NS % STEP == 0 && 4 % NK == 0, "whole steps");
      read(0, kf[0]);
#pragma unroll
      for (int s = 0; s < NS / STEP; ++s) {
        if (s + 1 < NS / STEP) read(s + 1, kf[(s + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < FR; ++u)
          st[u % NK] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[s & 1][u], qf[s * STEP + u / NK], st[u % NK], 0, 0, 0);
      }
    }
    settle(st);
    reads_done<KW == 1>();
    fetch(p.l.k, kt, blk + KW, page);
    // ---- the online softmax of the lane's row: the reference point of its exponentials moves when the
    // maximum has grown by more than 8 binary orders (probabilities up to 2^8 do no harm, and the
    // final division takes them out)
    float mx = -DM_INF;
    const int lim = min(vis, k1);  // (the shared part may end inside a block)
    bool masked = false;
    if constexpr (EDGE) masked = __builtin_amdgcn_ballot_w64(key0 + BK > lim) != 0;
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
    wait_loads<A::LOADS, KW == 1>();
    // A key that one row of the tile sees and another does not: its probability is 0 there, but 0
    // times a value that is no finite number is none. Blocks with such keys (the last of a sequence)
    // are looked through. If there is one, the product leaves out what is not finite, and that is added
    // key by key to the rows that see it; the other rows keep their bits.
    bool odd = false;
    if (EDGE && masked && __builtin_amdgcn_ballot_w64(vis > 0 && vis < min(key0 + BK, k1)) != 0) {
      uint32_t bad = 0;
#pragma unroll 1
      for (int i = lane; i < TILE / 16; i += 64) {
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(vt + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= ((w[e] & 0x7f80u) == 0x7f80u) | ((w[e] & 0x7f800000u) == 0x7f800000u);
      }
      odd = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
    }
    // ---- O^T += V^T P^T
    auto product = [&](auto only_finite) {
      constexpr bool FINITE = decltype(only_finite)::value;
      constexpr int KG = BK == 16 ? 1 : 2;  // groups of four keys a lane has of a fragment
      // Pairs of probabilities: the next number below, cut to bf16, and what that leaves of each, rounded to bf16; a
      // product each, so that a probability counts to 2^-16 of itself. (Below, so that neither part of a probability
      // above zero is zero: times an infinite value that would be no number, where the result is infinite. The first part
      // alone, 2^-8: 201 us for 215 at 2048 rows behind 32768 keys, 41.4 for 44.6 at 512 rows behind 16256, 1 %
      // where rows are few; the result's error against 64 bits was 2.2e-3 where its own rounding to bf16 makes 1.66e-3.)
      uint32_t pb[2][BK / 8];
#pragma unroll
      for (int i = 0; i < BK / 8; ++i) {
        const float p0 = st[i >> 1][2 * (i & 1)], p1 = st[i >> 1][2 * (i & 1) + 1];
        const uint32_t w0 = __builtin_elementwise_sub_sat(__float_as_uint(p0), 1u), w1 = __builtin_elementwise_sub_sat(__float_as_uint(p1), 1u);
        pb[0][i] = __builtin_amdgcn_perm(w1, w0, 0x07060302);
        pb[1][i] = dm_f2bf2(p0 - __uint_as_float(w0 & 0xffff0000u), p1 - __uint_as_float(w1 & 0xffff0000u));
      }
      s16x4_t vf[2][4][KG];
      constexpr int BATCHES = NK / KG * NC / 4;  // of four fragments
      auto read = [&](int b, s16x4_t (&f)[4][KG]) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int h = 0; h < KG; ++h) {
            const int t = (4 * b + u) % NC, kg = (4 * b + u) / NC, key = 16 * KG * kg + 16 * h + 4 * lg + (l16 >> 2);
            typedef __attribute__((address_space(3))) s16x4_t lds4;
            f[u][h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(vt + key * ROWB + ((t ^ A::swz(key)) << 5) + 8 * (l16 & 3)));
            if constexpr (FINITE) {
#pragma unroll
              for (int e = 0; e < 4; ++e) f[u][h][e] = (f[u][h][e] & 0x7f80) == 0x7f80 ? (short)0 : f[u][h][e];
            }
          }
      };
      read(0, vf[0]);
#pragma unroll
      for (int b = 0; b < BATCHES; ++b) {
        if (b + 1 < BATCHES) read(b + 1, vf[(b + 1) & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int t = (4 * b + u) % NC, kg = (4 * b + u) / NC;
            if constexpr (KG == 1) {
              const s16x4_t pv = __builtin_bit_cast(s16x4_t, u32x2_t{pb[part][0], pb[part][1]});
              o[t] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(vf[b & 1][u][0], pv, o[t], 0, 0, 0);
            } else {
              const bf16x8_t v = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(vf[b & 1][u][0], vf[b & 1][u][KG - 1], 0, 1, 2, 3, 4, 5, 6, 7));
              const bf16x8_t pv =
                  __builtin_bit_cast(bf16x8_t, u32x4_t{pb[part][4 * kg], pb[part][4 * kg + 1], pb[part][4 * kg + 2], pb[part][4 * kg + 3]});
              o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pv, o[t], 0, 0, 0);
            }
          }
      }
    };
    if constexpr (!EDGE) {
      product(std::false_type{});
    } else if (!odd) {
      product(std::false_type{});
    } else {
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
      product(std::true_type{});
    }
    reads_done<KW == 1>();
    fetch(p.l.v, vt, blk + KW, page);
  };
  int turn = 0;
#pragma unroll 1
  for (; turn < whole; ++turn) one_block(turn, std::false_type{});
#pragma unroll 1
  for (; turn < turns; ++turn) one_block(turn, std::true_type{});
  };
  walk(lds + set * 2 * TILE, lds + set * 2 * TILE + TILE);
  wait_loads<0, false>();  // (the last turns' requests write zeros: not into the LDS of whoever comes next)
  l_i = l_i + dm_xor_lane<16>(l_i);
  l_i = l_i + dm_xor_lane<32>(l_i);

  int t_lo = 0;  // the first of the channel tiles that this wavefront goes on with
  if constexpr (KW > 1) {
    // the wavefronts' sums meet: each leaves its own in LDS and takes a share of the channels of all
    static_assert(NC % KW == 0, "whole channel tiles a wavefront");
    __syncthreads();
    f32x4_t* const ob = reinterpret_cast<f32x4_t*>(lds);
    float2* const ml = reinterpret_cast<float2*>(lds + (size_t)KW * 16 * HD * 4);
#pragma unroll
    for (int t = 0; t < NC; ++t) ob[(set * NC + t) * 64 + lane] = o[t];
    if (lg == 0) ml[set * 16 + l16] = make_float2(m_i, l_i);
    __syncthreads();
    float w[KW], m = -DM_INF, l = 0.f;
#pragma unroll
    for (int s = 0; s < KW; ++s) m = fmaxf(m, ml[s * 16 + l16].x);
#pragma unroll
    for (int s = 0; s < KW; ++s) {
      const float2 v = ml[s * 16 + l16];
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
        const f32x4_t v = ob[(s * NC + t_lo + u) * 64 + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = dm_fma(v[e], w[s], sum[e]);
      }
      o[u] = sum;
    }
  }
  if (rho >= rows) return;
  constexpr int NT = KW > 1 ? NC / KW : NC;
  if (finishes) {
#pragma unroll
    for (int u = 0; u < NT; ++u) store_result<HD>(p, row_head, 16 * (t_lo + u) + 4 * lg, o[u], l_i, vis > 0);
    return;
  }
  const size_t at = (size_t)((SHARED ? 0 : p.chunks[0]) + chunk) * p.b.B * p.T * p.Hq + row_head;
#pragma unroll
  for (int u = 0; u < NT; ++u) *reinterpret_cast<f32x4_t*>(p.part_o + at * HD + 16 * (t_lo + u) + 4 * lg) = o[u];
  if (lg == 0 && t_lo == 0) p.part_ml[at] = make_float2(m_i, l_i);
}

template <int HD>
constexpr int attend_lds() {
  constexpr int wide = Attend<HD, 4, 64>::LDS, narrow = Attend<HD, 1, 16>::LDS;
  return wide > narrow ? wide : narrow;
}

// What it measured, 16 query heads on 2 KV heads of 256, shared keys / own keys a sequence, both forms in one launch:
//   2048 rows (64 sequences of 4 tokens x 8 heads), 32768 / 512   202-242 us by the card's clock, 570-690 TFLOP/s
//   512 rows (16 x 4 x 8), 16256 / 77                             38 us, 450 TFLOP/s
//   64 rows (8 x 1 x 8), 6592 / 200                               13-14 us, where a copy of its 16 MB takes 3.3
//   8 rows a sequence, nothing shared: one of 32768 keys 14-15 us, 4.5 TB/s; 8 of 4000-8000 19 us, 64 of 750-1500 25 us, 5 TB/s and more
// Wide: the matrix cores are busy for 47 % of the time (38 % at 512 rows), LDS a third (V's transposing reads run at half the
// rate of K's), 38 % of the wavefronts' cycles are waits, most of them at the four barriers a block: K's tile and V's have
// arrived, K's and V's may be written again. With one part of each probability alone, 185 us became 140 with the fetches
// taken out and 152 with V's reads; the softmax was within the noise. Larger tiles (128 rows, each
// fragment of K and V for two products) were 188-195 us with twice the partial sums, 32 x 32 products slower.
// At a width of 256 the wide forms have 256 registers, and 29 and 56 of them in scratch memory: around and in
// the loop of blocks with masks, none in the loop of full blocks.
// Narrow: a chain of trips to memory, table, keys, values a turn; a workgroup has as much in flight as LDS holds.
// Workgroups below `split` have chunks of the shared part, the others of the sequences' own.
template <int HD, bool WIDE_SHARED, bool WIDE_OWN>
__global__ __launch_bounds__(64 * kWaves, 2) void attend_kernel(PagedArgs p, int split) {
  __shared__ __align__(1024) unsigned char lds[attend_lds<HD>()];
  __shared__ uint32_t ids[kChunkPages];
  if ((int)blockIdx.x < split) attend_part<HD, WIDE_SHARED ? 4 : 1, WIDE_SHARED ? 64 : 16, true>(p, blockIdx.x, lds, ids);
  else attend_part<HD, WIDE_OWN ? 4 : 1, WIDE_OWN ? 64 : 16, false>(p, blockIdx.x - split, lds, ids);
}

// 42 MB in 13.5 us (3.1 TB/s) at 2048 rows in 10 slots, 35 MB in 9 us (3.9 TB/s) at 512 rows in 33, 4 us (a launch and two
// trips) where there are few rows, 10 us for 8 rows in 171 slots. A chain of trips: lengths, then a wavefront's share of the
// slots at once, then LDS; at 10 slots a wavefront has two or three loads in flight, and 56 % of the wavefronts' cycles
// are waits. More wavefronts a row were slower from 512 rows on.
// Joins the slots of a (row, head): four channels a lane, the slots dealt to the wavefronts, whose sums
// meet in LDS. Chunks past what the row sees were not computed for it, or hold nothing of it, and are
// not read. A slot of weight 0 is added like the others: a value in it that is not finite makes no number
// of the channel, as it does beside the row's maximum.
constexpr int kJoinWaves = 4;
template <int HD>
__global__ __launch_bounds__(64 * kJoinWaves) void join_kernel(PagedArgs p) {
  constexpr int LANES = HD / 4, PARTS = 64 * kJoinWaves / LANES;
  __shared__ float4 so[PARTS][LANES];
  __shared__ float2 sml[PARTS];
  const int r = blockIdx.y, head = blockIdx.x, part = threadIdx.x / LANES, ch = 4 * (threadIdx.x % LANES), seq = r / p.T;
  const int vis = batch_len(p.b, seq) - p.T + (r - seq * p.T) + 1;
  const size_t row_head = (size_t)r * p.Hq + head, slot = (size_t)p.b.B * p.T * p.Hq;
  const int ns = vis > 0 ? min(p.chunks[0], (vis + p.chunk[0] - 1) / p.chunk[0]) : 0;
  const int no = vis > p.shared ? min(p.chunks[1], (vis - p.shared + p.chunk[1] - 1) / p.chunk[1]) : 0;
  auto place = [&](int i) { return (size_t)(i < ns ? i : p.chunks[0] + i - ns) * slot + row_head; };
  // the slots of this part, eight at a time (few turns: each waits for memory): a running maximum as over keys
  float m = -DM_INF, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = part; i0 < ns + no; i0 += 8 * PARTS) {
    float2 v[8];
    f32x4_t x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u * PARTS;
      v[u] = make_float2(-DM_INF, 0.f);
      x[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (i < ns + no) {
        v[u] = p.part_ml[place(i)];
        x[u] = *reinterpret_cast<const f32x4_t*>(p.part_o + place(i) * HD + ch);
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (i0 + u * PARTS >= ns + no) continue;
      const float mn = fmaxf(m, v[u].x);
      const float a = m > -DM_INF ? __builtin_amdgcn_exp2f((m - mn) * p.c2) : 1.f;  // (nothing yet, or NaN, which stays)
      const float w = v[u].x > -DM_INF ? __builtin_amdgcn_exp2f((v[u].x - mn) * p.c2) : v[u].y != v[u].y ? 1.f : 0.f;
      m = mn;
      l = dm_fma(v[u].y, w, l * a);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = dm_fma(x[u][e], w, o[e] * a);
    }
  }
  so[part][ch / 4] = make_float4(o[0], o[1], o[2], o[3]);
  if (ch == 0) sml[part] = make_float2(m, l);
  __syncthreads();
  if (part) return;
  float mt = -DM_INF;
#pragma unroll
  for (int q = 0; q < PARTS; ++q) mt = fmaxf(mt, sml[q].x);
  l = 0.f;
  o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < PARTS; ++q) {
    const float2 v = sml[q];
    const float4 x = so[q][ch / 4];
    const float w = v.x > -DM_INF ? __builtin_amdgcn_exp2f((v.x - mt) * p.c2) : v.y != v.y ? 1.f : 0.f;
    l = dm_fma(v.y, w, l);
    o[0] = dm_fma(x.x, w, o[0]);
    o[1] = dm_fma(x.y, w, o[1]);
    o[2] = dm_fma(x.z, w, o[2]);
    o[3] = dm_fma(x.w, w, o[3]);
  }
  store_result<HD>(p, row_head, ch, o, l, vis > 0);
}

template <int HD>
int attend(ornith_ctx* ctx, PagedArgs a, int max_rows) {
  const int own_rows = a.T * (a.Hq / a.l.Hkv), shared_rows = a.b.B * own_rows;
  // Wide from more than 128 rows: below, the tiles of 16 rows read their keys out of the die's cache often
  // enough, and their chunks are longer, so that less goes through memory. Both launches, us, narrow / wide,
  // at 2000 / 6600 / 16300 keys: 2 KV heads of 256, 64 rows 11.2 / 13.4, 16.2 / 17.6, 22.6 / 23.4; 128 rows 11.8 / 14.6, 19.7 / 21.8,
  // 26.1 / 31.9; 192 rows 15.0 / 15.8, 23.0 / 25.5, 36.0 / 34.2; 256 rows 16.4 / 17.7, 25.4 / 27.2, 33.6 / 35.0; 512 rows
  // 21.6 / 22.3, 30.4 / 29.9, 52.3 / 43.4. 8 KV heads of 128: 128 rows 14.5 / 16.1, 20.1 / 22.3; 192 rows 19.8 / 20.1, 26.0 / 25.7; 256 rows
  // 21.0 / 22.4, 30.1 / 28.8. 2 KV heads of 128: 192 rows 10.8 / 11.5, 14.4 / 18.0; 384 rows 13.5 / 13.3, 19.4 / 21.1. One of 64: 256 rows
  // 8.7 / 9.2, 10.4 / 10.7, 512 rows 10.0 / 10.2, 12.1 / 14.3: few heads, or narrow ones, could stay narrow for longer.
  const bool wide[2] = {shared_rows > 128, own_rows > 128};
  int64_t grid[2];
  const int keys[2] = {a.shared, max_rows - a.shared}, rows[2] = {shared_rows, own_rows}, seqs[2] = {1, a.b.B};
  for (int part = 0; part < 2; ++part) {
    // chunks: two workgroups for every compute unit (both launches, us, one / one and a half / two / three a
    // unit: 2 KV heads of 256, 512 rows at 16300 keys 44.6 / 44.5 / 46.7 / 51.4, 2048 at 32768 325 / 260 / 217 / 260; 8 of 128, 1024 rows at 8200
    // 100 / 85 / 76 / 81; one of 64, 2048 rows at 16300 36 / 35.4 / 32.1 / 33; but 64 rows of 2 of 256 at 6600 13.6 / 17 / 16.9 / 17: with one
    // each, a unit is done once); whole blocks of
    // 64 (a chunk that begins inside a page touches one page more than it has). None is shorter than 128 keys,
    // 192 in the narrow form: with more of them the sums that go through memory cost more than the keys'
    // reads gain (at least 64 / 128 / 192 / 256 keys, us: wide, 512 rows of 2 KV heads of 256 at 2000 keys 29.3 / 21.2 / 21.2 / 21.9, 256
    // rows 22.9 / 17.7 / 17.4 / 18.1; narrow, 32 rows of 8 of 128 at 2000 12.4 / 10.3 / 9.7 / 9.6, 32 of 2 of 256 at 1000 10 / 10.1 / 10.5 / 10.8,
    // 64 of 2 of 256 at 6600 18.2 / 18.2 / 17.1 / 13.8, 64 of one of 64 at 6600 9.8 / 8.7 / 8.9 / 8.9).
    const int tile = wide[part] ? 64 : 16, most = ((kChunkPages - 1) << a.l.shift) / 64 * 64;
    const int64_t tiles = (rows[part] + tile - 1) / tile, pairs = (int64_t)seqs[part] * a.l.Hkv;
    const int64_t want = std::max<int64_t>(1, (2 * ctx->compute_units + tiles * pairs - 1) / (tiles * pairs));
    const int len = (int)std::min<int64_t>(std::max<int64_t>(wide[part] ? 128 : 192, ((keys[part] + want - 1) / want + 63) / 64 * 64), most);
    a.chunk[part] = len;
    a.chunks[part] = (keys[part] + len - 1) / len;
    grid[part] = (a.chunks[part] * pairs + kDies - 1) / kDies * kDies * tiles;
  }
  if (a.chunks[0] + a.chunks[1] == 0) {  // max_rows is 0: no row sees anything
    a.chunks[1] = 1;
    grid[1] = ((int64_t)a.b.B * a.l.Hkv + kDies - 1) / kDies * kDies * ((own_rows + (wide[1] ? 63 : 15)) / (wide[1] ? 64 : 16));
  }
  ORN_REQUIRE(grid[0] + grid[1] < int64_t(1) << 24, "sdpa_paged: %lld workgroups", (long long)(grid[0] + grid[1]));  // (2^32 threads a launch)
  const int slots = a.chunks[0] + a.chunks[1];
  const size_t cells = (size_t)a.b.B * a.T * a.Hq;
  if (slots != 1) {
    void* base = nullptr;
    if (int rc = ornith_scratch(ctx, slots * cells * (HD * 4 + 8) + 512, &base)) return rc;
    ScratchCursor sc(base);
    a.part_o = sc.take<float>(slots * cells * HD);
    a.part_ml = sc.take<float2>(slots * cells);
  }
  // (the shared part has all sequences' rows: it is wide where a sequence's own part is)
  void (*const kernel)(PagedArgs, int) =
      wide[1] ? attend_kernel<HD, true, true> : wide[0] ? attend_kernel<HD, true, false> : attend_kernel<HD, false, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(grid[0] + grid[1])), dim3(64 * kWaves), 0, ctx->stream, a, (int)grid[0]);
  ORN_LAUNCH_CHECK("attend_kernel");
  if (slots != 1) {
    hipLaunchKernelGGL(join_kernel<HD>, dim3(a.Hq, a.b.B * a.T), dim3(64 * kJoinWaves), 0, ctx->stream, a);
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
  const float c2 = scale * 1.44269504088896341f;
  ORN_REQUIRE(scale > 0.f && c2 < DM_INF, "sdpa_paged: scale %g", scale);
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
  a.c2 = c2;
  switch (pages->hd) {
    case 64: return attend<64>(ctx, a, batch->max_rows);
    case 128: return attend<128>(ctx, a, batch->max_rows);
    default: return attend<256>(ctx, a, batch->max_rows);
  }
}

}  // extern "C"
