// Log probabilities of given tokens, with the row's logsumexp, entropy and most probable
// alternatives. No counterpart in the reference, whose samplers keep their log-softmax to
// themselves (/root/reference/src/sample.rs:205-225); greedy_rows beside it returns the token.
//
// With m = max x, L = sum e^(x - m), S = sum e^(x - m) (x - m) over a row:
//   lse = m + ln L      log p(t) = (x_t - m) - ln L      H = ln L - S / L
// (x_t - m before the logarithm is taken off, so that a sure token's near-zero result keeps its
// digits). All sums are fp32 over fp32 values.
#include "dmath.h"
#include "rt.h"

#include <algorithm>

namespace {

constexpr int kMaxTop = 32;  // alternatives a row

// Two launches. The first reads the logits once: a row is cut into groups of contiguous tokens, a
// wavefront takes some groups one after another and leaves its (m, L, S) and every group's best value.
// The second, a workgroup a row, joins the sums; and as the k best tokens of a row lie in its k best
// groups (by best value, then by place: each of k better groups holds a token that comes before any of
// the group's), it looks through those alone, and in them, for the same reason, at the k best 16-byte
// pieces.
constexpr int kFinish = 1024;                // threads of the second launch
constexpr int kPass = 4;                     // passes of so many threads over a row's groups, or over the pieces of the best ones
constexpr int kGroups = kPass * kFinish;     // groups a row at most
constexpr int kGroupPieces = 128;            // 16-byte pieces a group: 2 KB, two loads a lane
static_assert(kMaxTop * kGroupPieces <= kPass * kFinish, "the best groups' pieces in as many passes");
constexpr int kCands = 256;                  // candidates that are ranked against each other
static_assert(kMaxTop * 8 <= kCands, "the best pieces' tokens among them");
constexpr int kMaxV = (kGroups * kGroupPieces - 1) * 4;  // logits a row: what fits kGroups groups of fp32 at any alignment
constexpr float kL2E = 1.44269502162933349609375f, kL2ELow = 1.925963033500e-8f, kLn2 = 0.693147180559945309f;
constexpr float kFloor = -200.f;             // e^kFloor is 0 in fp32: differences stop there, so that -inf makes no NaN

struct LogprobArgs {
  const void* x;
  const uint32_t* tokens;  // [rows, n_tokens]
  float* logprobs;         // [rows, n_tokens]
  float* entropy;          // [rows]
  float* lse;              // [rows]
  uint32_t* top_ids;       // [rows, k]
  float* top_logprobs;     // [rows, k]
  float4* sums;            // [rows, runs]: m, L without its terms of 1, S, and what rounding the exponents took from L
  float* ones;             // [rows, runs]: how many terms of L are 1 (the maximum's)
  uint32_t* best;          // [rows, groups]: order of the best value
  int64_t stride;
  int V, n_tokens, k;
  int groups, run, runs;   // groups a row; groups a wavefront takes; wavefronts a row
};

// A value's place among all: larger for a larger value, -0 and 0 the same, NaN below everything.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0u : v == 0.f ? 0x80000000u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A row as 16-byte pieces at 16-byte addresses: piece j holds tokens [PER j - head, + PER). The first
// piece may begin before the row (in the 16 bytes that hold its first token) and the last end behind
// it: what is no token of the row is told apart by its number, and nothing behind the piece that
// holds the last one is read.
template <bool F32>
struct Row {
  static constexpr int PER = F32 ? 4 : 8, ES = F32 ? 4 : 2;
  const unsigned char* base;  // of token 0
  __amdgpu_buffer_rsrc_t buf;
  int V, head;
  __device__ __forceinline__ Row(const LogprobArgs& p, size_t row) {
    base = static_cast<const unsigned char*>(p.x) + (size_t)(row * p.stride) * ES;
    V = p.V;
    head = (int)((uintptr_t)base & 15) / ES;
    buf = dm_buffer(base - head * ES, ((V + head) * ES + 3) & ~3);
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (F32) return reinterpret_cast<const float*>(base)[i];
    return dm_bf2f(reinterpret_cast<const bf16_t*>(base)[i]);
  }
  __device__ __forceinline__ int first(int piece) const { return PER * piece - head; }
  __device__ __forceinline__ bool has(int t) const { return (unsigned)t < (unsigned)V; }
  __device__ __forceinline__ void load(int piece, float (&x)[PER]) const {
    const dm_u32x4 w = __builtin_bit_cast(dm_u32x4, __builtin_amdgcn_raw_buffer_load_b128(buf, 16 * piece, 0, 0));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (F32) {
        x[i] = __uint_as_float(w[i]);
      } else {
        x[2 * i] = dm_bf2f_lo(w[i]);
        x[2 * i + 1] = dm_bf2f_hi(w[i]);
      }
    }
  }
};

// The terms e^0 = 1 of L are counted apart (N): next to them the others would lose their last digits, and a
// sure token's log probability is made of those.
// (m, L, S, C, N) of two parts as one: S follows the reference point, e^(x - m') (x - m') = f (e^(x - m) (x - m) + e^(x - m) (m - m')).
__device__ __forceinline__ void move_to(float m_new, float& m, float& l, float& s, float& c, float& n) {
  const float d = __builtin_elementwise_maximum(m - m_new, kFloor), f = dm_exp(d);  // (m = -inf: nothing there yet, or NaN, which stays)
  l += n;
  n = 0.f;
  s = f * dm_fma(l, d, s);
  l *= f;
  c *= f;
  m = m_new;
}

// Bound by the logits' stream: 700 rows of 248320 bf16 (348 MB) take 69-76 us, 4.6-5.0 TB/s, as a copy; four
// tenths of its wavefronts' cycles are waits for memory, and the exponentials hide behind them. One row takes
// 3.2 us, a launch's worth; 350 rows of fp32 (348 MB) 61-65 us, 5.3-5.7 TB/s.
// grid (runs of groups / 4, rows)
template <bool F32>
__global__ __launch_bounds__(256) void logprobs_sum_kernel(LogprobArgs p) {
  using R = Row<F32>;
  constexpr int PER = R::PER;
  const int lane = threadIdx.x & 63, w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t row = blockIdx.y;
  if (w >= p.runs) return;
  const R r(p, row);
  const int g_end = min(p.groups, (w + 1) * p.run);
  float m = -DM_INF, l = 0.f, s = 0.f, c = 0.f, n = 0.f;
  for (int g = w * p.run; g < g_end; ++g) {
    float x[2][PER];
    const int piece = g * kGroupPieces + lane;
    r.load(piece, x[0]);
    r.load(piece + 64, x[1]);
    if (r.first(g * kGroupPieces) < 0 || r.first((g + 1) * kGroupPieces) > p.V) {  // the row's first group or its last
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < PER; ++i) x[u][i] = r.has(r.first(piece + 64 * u) + i) ? x[u][i] : -DM_INF;
    }
    float best = -DM_INF;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < PER; ++i) best = fmaxf(best, x[u][i]);
    best = dm_wave_max<64>(best);
    bool low = false;
    if (best == -DM_INF) {  // masked tokens or NaN only: which of them
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int t = r.first(piece + 64 * u) + i;
          low = low || (r.has(t) && x[u][i] == -DM_INF);
        }
    }
    if (best > m) move_to(best, m, l, s, c, n);
    if (best == m && __builtin_fabsf(m) < DM_INF) {  // (few groups hold the maximum so far; no distribution has an infinite one)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          n += x[u][i] == m ? 1.f : 0.f;
          x[u][i] = x[u][i] == m ? -DM_INF : x[u][i];
        }
    }
    const float ref = m > -DM_INF ? m : 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        // e^d = 2^t (1 + ln2 (lo + d kL2ELow)): t is rounded at its own size, and what that takes is put
        // back in the sum (C), or a sure token's probability would carry the error of far smaller ones
        const float d = __builtin_elementwise_maximum(x[u][i] - ref, kFloor);
        const float t = d * kL2E, lo = dm_fma(d, kL2E, -t);
        const float e = __builtin_amdgcn_exp2f(t);
        l += e;
        s = dm_fma(e, d, s);
        c = dm_fma(e, lo, c);
      }
    if (p.k) {
      uint32_t o = order_of(best);
      if (best == -DM_INF && __builtin_amdgcn_ballot_w64(low) == 0) o = 0;
      if (lane == 0) p.best[row * p.groups + g] = o;
    }
  }
  l = dm_wave_sum<64>(l);
  s = dm_wave_sum<64>(s);
  c = dm_wave_sum<64>(c);
  n = dm_wave_sum<64>(n);
  if (lane == 0) {
    p.sums[row * p.runs + w] = make_float4(m, l, s, c);
    p.ones[row * p.runs + w] = n;
  }
}

// The value that order_of made `o` of (-0 as 0, any NaN as one).
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == 0 ? __builtin_nanf("") : __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

struct Select {
  uint32_t key[kPass * kFinish];
  uint32_t range[kFinish / 64][2];
  uint32_t counts[2][kFinish / 64][2];
  int list[kMaxTop], found[64], n;
  uint32_t least;
};

// the value of lane l ^ S, and what the lanes of a wavefront (W = 64) or of a row of 16 come to
template <int S>
__device__ __forceinline__ uint32_t other(uint32_t v) { return __float_as_uint(dm_xor_lane<S>(__uint_as_float(v))); }
template <int W, class Op>
__device__ __forceinline__ uint32_t all_lanes(uint32_t v, Op op) {
  if constexpr (W == 64) {
    v = op(v, other<32>(v));
    v = op(v, other<16>(v));
  }
  v = op(v, other<8>(v));
  v = op(v, other<4>(v));
  v = op(v, other<2>(v));
  return op(v, other<1>(v));
}

// The k best of sh.key[0 .. n), n >= k, equal ones by the lower number, their numbers into sh.list, best
// first; returns the least of them. The workgroup counts, two bits of a bound a turn, how
// many keys reach it; it starts below what the largest and the smallest have in common and is done as
// soon as that are no more than a wavefront has lanes: those are ranked. More equal keys than that at the bound are
// cut the same way by their numbers. (Loops stay loops here: a launch of one workgroup takes as long
// as its code takes to arrive.)
__device__ __forceinline__ uint32_t select_best(int n, int k, Select& sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto add = [](uint32_t a, uint32_t b) { return a + b; };
  auto larger = [](uint32_t a, uint32_t b) { return max(a, b); };
  uint32_t hi = 0, lo = 0;  // of the keys, and of their complements
#pragma unroll 1
  for (int i = tid; i < n; i += kFinish) {
    hi = max(hi, sh.key[i]);
    lo = max(lo, ~sh.key[i]);
  }
  hi = all_lanes<64>(hi, larger);
  lo = all_lanes<64>(lo, larger);
  if (lane == 0) {
    sh.range[wave][0] = hi;
    sh.range[wave][1] = lo;
  }
  if (tid == 0) sh.n = 0;
  __syncthreads();
  hi = all_lanes<16>(sh.range[lane & 15][0], larger);
  lo = ~all_lanes<16>(sh.range[lane & 15][1], larger);
  const uint32_t same = hi ^ lo;
  int have = n, bit = same ? (31 - __builtin_clz(same)) & ~1 : -2;  // pairs of bits from the one that holds the first difference
  uint32_t bound = bit < 0 ? lo : bit == 30 ? 0 : hi >> (bit + 2) << (bit + 2), edge = 0;
  bool by_number = false;
  auto value = [&](int i) {
    const uint32_t v = i < n ? sh.key[i] : 0;
    return !by_number ? v : v > edge ? 0x2000u : v == edge && i < n ? 0x1fffu - i : 0u;
  };
  static_assert(kPass * kFinish <= 0x1000, "numbers in twelve bits");
  int turn = 0;
#pragma unroll 1
  for (;;) {
    if (have <= 64 || bit < 0) {
      if (have <= 64) break;  // (numbers are all different: cut by them, 64 is reached)
      by_number = true;
      edge = bound;
      bound = 0;
      bit = 12;
    }
    const uint32_t one = bound | 1u << bit, two = bound | 2u << bit, three = bound | 3u << bit;
    int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll 1
    for (int i = wave * 64; i < n; i += kFinish) {
      const uint32_t v = value(i + lane);
      c1 += __popcll(__builtin_amdgcn_ballot_w64(v >= one));
      c2 += __popcll(__builtin_amdgcn_ballot_w64(v >= two));
      c3 += __popcll(__builtin_amdgcn_ballot_w64(v >= three));
    }
    if (lane == 0) {
      sh.counts[turn][wave][0] = (uint32_t)c1 | (uint32_t)c2 << 16;  // (at most kPass * kFinish each)
      sh.counts[turn][wave][1] = (uint32_t)c3;
    }
    __syncthreads();  // (the other turn's counts have been read by all when this one's are complete)
    const uint32_t a = all_lanes<16>(sh.counts[turn][lane & 15][0], add);
    const int n1 = (int)(a & 0xffff), n2 = (int)(a >> 16), n3 = (int)all_lanes<16>(sh.counts[turn][lane & 15][1], add);
    const int t = n3 >= k ? 3 : n2 >= k ? 2 : n1 >= k ? 1 : 0;
    bound |= (uint32_t)t << bit;
    if (t) have = t == 3 ? n3 : t == 2 ? n2 : n1;
    bit -= 2;
    turn ^= 1;
  }
#pragma unroll 1
  for (int i = tid; i < n; i += kFinish)
    if (value(i) >= bound) sh.found[atomicAdd(&sh.n, 1)] = i;
  __syncthreads();
  // every wavefront has all of them in its lanes and ranks its share
  const int mine = lane < have ? sh.found[lane] : 0;
  const uint32_t v = lane < have ? sh.key[mine] : 0;
#pragma unroll 1
  for (int e = wave; e < have; e += kFinish / 64) {
    const int i = __builtin_amdgcn_readlane(mine, e);
    const uint32_t iv = (uint32_t)__builtin_amdgcn_readlane((int)v, e);
    const int rank = __popcll(__builtin_amdgcn_ballot_w64(lane < have && (v > iv || (v == iv && mine < i))));
    if (lane == 0 && rank < k) {
      sh.list[rank] = i;
      if (rank == k - 1) sh.least = iv;
    }
  }
  __syncthreads();
  return sh.least;
}

// A chain of latencies: the sums and the groups' best values, four to six turns of the count, the best groups'
// logits, a rank. 9.2 us for one row with twenty alternatives of 248320, 6.4 us for four rows with five of 32768
// (f32), 19 us for 700 rows with eight, two workgroups of 1024 a compute unit. (17.6 and 32 with a selection
// that was unrolled and cut by one bit a turn: with one workgroup the code's own way in counts.)
// grid (rows)
template <bool F32>
__global__ __launch_bounds__(kFinish) void logprobs_finish_kernel(LogprobArgs p) {
  using R = Row<F32>;
  constexpr int PER = R::PER, SHIFT = F32 ? 0 : 16;  // (a bf16's order is in its upper half)
  __shared__ float4 red[kFinish / 64];
  __shared__ float red_n[kFinish / 64];
  __shared__ Select sel;
  __shared__ int groups[kMaxTop], n_cands;
  __shared__ uint32_t cand_o[kCands], cand_i[kCands];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.x;
  const R r(p, row);

  // everything that does not wait for something else is asked for first
  float4 part = make_float4(-DM_INF, 0.f, 0.f, 0.f);
  float n1 = 0.f;
  if (tid < p.runs) {  // (runs <= the workgroup)
    part = p.sums[row * p.runs + tid];
    n1 = p.ones[row * p.runs + tid];
  }
  if (p.k)
#pragma unroll 1
    for (int i = tid; i < p.groups; i += kFinish) sel.key[i] = p.best[row * p.groups + i] >> SHIFT;
  float asked = -DM_INF;
  if (tid < p.n_tokens) {
    const uint32_t t = p.tokens[row * p.n_tokens + tid];
    if (t < (uint32_t)p.V) asked = r.at(t);
  }
  if (tid == 0) n_cands = 0;
  // the row's sums
  const float wm = dm_wave_max<64>(part.x);
  if (part.x < wm) move_to(wm, part.x, part.y, part.z, part.w, n1);
  part = make_float4(wm, dm_wave_sum<64>(part.y), dm_wave_sum<64>(part.z), dm_wave_sum<64>(part.w));
  n1 = dm_wave_sum<64>(n1);
  if (lane == 0) {
    red[wave] = part;
    red_n[wave] = n1;
  }
  __syncthreads();
  part = red[lane & 15];
  n1 = red_n[lane & 15];
  const float m = dm_wave_max<16>(part.x);
  if (part.x < m) move_to(m, part.x, part.y, part.z, part.w, n1);
  const float s = dm_row_sum(part.z), rest = dm_fma(kLn2, dm_fma(kL2ELow, s, dm_row_sum(part.w)), dm_row_sum(part.y));
  n1 = dm_row_sum(n1);
  // L = l + low, the sum and what its rounding left; ln L = ln l + low / l
  const float l = n1 + rest, back = l - n1, low = (n1 - (l - back)) + (rest - back);
  const float ref = m > -DM_INF ? m : 0.f;
  const bool none = l == 0.f;
  const float logl = none ? 0.f : dm_log(l) + low / l;
  if (tid == 0) {
    if (p.lse) p.lse[row] = none ? -DM_INF : ref + logl;
    if (p.entropy) p.entropy[row] = none ? 0.f : logl - s / l;
  }
  for (int i = tid; i < p.n_tokens; i += kFinish) {
    if (i != tid) {
      const uint32_t t = p.tokens[row * p.n_tokens + i];
      asked = t < (uint32_t)p.V ? r.at(t) : -DM_INF;
    }
    p.logprobs[row * p.n_tokens + i] = (asked - ref) - logl;
  }
  if (p.k == 0) return;

  // the best groups
  const int kg = min(p.k, p.groups), np = kg * kGroupPieces;
  uint32_t least = select_best(p.groups, kg, sel);
  if (tid < kg) groups[tid] = sel.list[tid];
  if (kg < p.k) least = 0;  // (fewer groups than alternatives: all of their tokens)
  __syncthreads();
  auto piece_of = [&](int i) { return groups[i / kGroupPieces] * kGroupPieces + i % kGroupPieces; };
  // their tokens that reach the bound of the groups: mostly not many more than k, and those are ranked
  {
    float next[PER];
    const int i_first = wave * 64;
    if (i_first < np) r.load(piece_of(i_first) + lane, next);
#pragma unroll 1
    for (int i0 = i_first; i0 < np; i0 += kFinish) {
      const int t0 = r.first(piece_of(i0) + lane);
      float x[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] = next[e];
      if (i0 + kFinish < np) r.load(piece_of(i0 + kFinish) + lane, next);
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const uint32_t o = order_of(x[e]);
        const uint64_t mask = __builtin_amdgcn_ballot_w64(r.has(t0 + e) && o >> SHIFT >= least);
        if (mask) {
          int at = 0;
          if (lane == 0) at = atomicAdd(&n_cands, __popcll(mask));
          at = __builtin_amdgcn_readfirstlane(at) + __popcll(mask & ((uint64_t(1) << lane) - 1));
          if ((mask >> lane & 1) && at < kCands) {
            cand_o[at] = o;
            cand_i[at] = t0 + e;
          }
        }
      }
    }
  }
  __syncthreads();
  const bool by_piece = n_cands > kCands;
  if (by_piece) {
    // Equal tokens without end, or many good ones in one group: the best pieces first. The groups in
    // ascending order, so that equal pieces are taken in the order of their tokens.
    if (wave == 0) {
      const int g = lane < kg ? sel.list[lane] : 0x7fffffff;
      int place = 0;
#pragma unroll 1
      for (int o = 0; o < kg; ++o) place += __builtin_amdgcn_readlane(g, o) < g;
      if (lane < kg) groups[place] = g;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < np; i += kFinish) {
      const int piece = piece_of(i);
      float x[PER];
      r.load(piece, x);
      uint32_t best = 0;
#pragma unroll
      for (int e = 0; e < PER; ++e) best = max(best, r.has(r.first(piece) + e) ? order_of(x[e]) >> SHIFT : 0u);
      sel.key[i] = best;
    }
    __syncthreads();
    least = select_best(np, p.k, sel);
  }
  if (by_piece) {
    // (the row has k tokens or more, but not always k pieces: then all of them)
    if (tid == 0) n_cands = 0;
    __syncthreads();
    if (tid < p.k * PER) {
      const int t = r.first(piece_of(sel.list[tid / PER])) + tid % PER;
      const uint32_t o = r.has(t) ? order_of(r.at(t)) : 0;
      if (r.has(t) && o >> SHIFT >= least) {
        const int at = atomicAdd(&n_cands, 1);
        cand_o[at] = o;
        cand_i[at] = t;
      }
    }
    __syncthreads();
  }
  const int n = n_cands;
  for (int i = wave; i < n; i += kFinish / 64) {
    const uint32_t o = cand_o[i], id = cand_i[i];
    int rank = 0;
    for (int j0 = 0; j0 < n; j0 += 64) {
      const int j = j0 + lane;
      rank += __popcll(__builtin_amdgcn_ballot_w64(j < n && (cand_o[j] > o || (cand_o[j] == o && cand_i[j] < id))));
    }
    if (lane == 0 && rank < p.k) {
      p.top_ids[row * p.k + rank] = id;
      p.top_logprobs[row * p.k + rank] = (value_of(o) - ref) - logl;
    }
  }
}

}  // namespace

extern "C" int ornith_token_logprobs(ornith_ctx* ctx, const void* d_logits, int dtype, int rows, int V, int64_t row_stride,
                                     const uint32_t* d_tokens, int n_tokens, int k, float* d_logprobs, float* d_entropy,
                                     float* d_lse, uint32_t* d_top_ids, float* d_top_logprobs) {
  ORN_REQUIRE(d_logits, "token_logprobs: null logits");
  ORN_REQUIRE(dtype == ORNITH_F32 || dtype == ORNITH_BF16, "token_logprobs: dtype %d", dtype);
  ORN_REQUIRE(rows >= 1 && rows <= 65535 && V >= 1 && row_stride >= V, "token_logprobs: rows=%d V=%d row_stride=%lld", rows, V, (long long)row_stride);
  ORN_REQUIRE(n_tokens >= 0 && (n_tokens == 0 || (d_tokens && d_logprobs)), "token_logprobs: %d tokens a row without their arrays", n_tokens);
  ORN_REQUIRE(n_tokens <= 1 << 30, "token_logprobs: %d tokens a row (at most 2^30)", n_tokens);  // (their numbers grow by a workgroup's threads)
  ORN_REQUIRE(k >= 0 && k <= kMaxTop && k <= V, "token_logprobs: %d alternatives of %d tokens (at most %d)", k, V, kMaxTop);
  ORN_REQUIRE(k == 0 || (d_top_ids && d_top_logprobs), "token_logprobs: alternatives without their arrays");
  ORN_REQUIRE(((uintptr_t)d_logits & (dtype == ORNITH_F32 ? 3 : 1)) == 0, "token_logprobs: misaligned logits");
  ORN_REQUIRE(V <= kMaxV, "token_logprobs: %d logits a row (at most %d)", V, kMaxV);
  ORN_REQUIRE(ctx, "token_logprobs: null context");
  const OrnDevice on(ctx);
  LogprobArgs p{};
  p.x = d_logits;
  p.tokens = d_tokens;
  p.logprobs = d_logprobs;
  p.entropy = d_entropy;
  p.lse = d_lse;
  p.top_ids = d_top_ids;
  p.top_logprobs = d_top_logprobs;
  p.stride = row_stride;
  p.V = V;
  p.n_tokens = n_tokens;
  p.k = k;
  const int per = dtype == ORNITH_F32 ? 4 : 8;
  const int64_t pieces = ((int64_t)V + 2 * per - 2) / per;  // at any alignment
  p.groups = (int)((pieces + kGroupPieces - 1) / kGroupPieces);
  // a wavefront takes one group while that fills the machine, eight where there are rows enough
  p.run = (int)std::min<int64_t>(8, std::max<int64_t>((p.groups + kFinish - 1) / kFinish, (int64_t)rows * p.groups / (32 * ctx->compute_units)));
  p.runs = (p.groups + p.run - 1) / p.run;
  void* base = nullptr;
  if (int rc = ornith_scratch(ctx, (size_t)rows * (p.runs * (sizeof(float4) + 4) + p.groups * 4) + 768, &base)) return rc;
  ScratchCursor sc(base);
  p.sums = sc.take<float4>((size_t)rows * p.runs);
  p.ones = sc.take<float>((size_t)rows * p.runs);
  p.best = sc.take<uint32_t>((size_t)rows * p.groups);
  const dim3 grid((p.runs + 3) / 4, rows);
  if (dtype == ORNITH_F32) hipLaunchKernelGGL(logprobs_sum_kernel<true>, grid, dim3(256), 0, ctx->stream, p);
  else hipLaunchKernelGGL(logprobs_sum_kernel<false>, grid, dim3(256), 0, ctx->stream, p);
  ORN_LAUNCH_CHECK("logprobs_sum_kernel");
  if (dtype == ORNITH_F32) hipLaunchKernelGGL(logprobs_finish_kernel<true>, dim3(rows), dim3(kFinish), 0, ctx->stream, p);
  else hipLaunchKernelGGL(logprobs_finish_kernel<false>, dim3(rows), dim3(kFinish), 0, ctx->stream, p);
  ORN_LAUNCH_CHECK("logprobs_finish_kernel");
  return ORNITH_OK;
}
