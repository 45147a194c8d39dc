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
// the group's), it looks through those alone.
constexpr int kGroups = 512;                 // groups a row at most
constexpr int kCands = 512;                  // candidates that are ranked against each other
constexpr int kFinish = 1024;                // threads of the second launch
constexpr float kL2E = 1.44269502162933349609375f, kL2ELow = 1.925963033500e-8f, kLn2 = 0.693147180559945309f;
constexpr float kFloor = -200.f;             // e^kFloor is 0 in fp32: differences stop there, so that -inf makes no NaN

typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

struct LogprobArgs {
  const void* x;
  const uint32_t* tokens;  // [rows, n_tokens]
  float* logprobs;         // [rows, n_tokens]
  float* entropy;          // [rows]
  float* lse;              // [rows]
  uint32_t* top_ids;       // [rows, k]
  float* top_logprobs;     // [rows, k]
  float4* sums;            // [rows, runs]: m, L, S, and what rounding the exponents took from L
  uint32_t* best;          // [rows, groups]: order of the best value
  int64_t stride;
  int V, n_tokens, k;
  int steps, groups, run, runs;  // loads a lane a group; groups a row; groups a wavefront takes; wavefronts a row
};

// A value's place among all: larger for a larger value, -0 and 0 the same, NaN below everything.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return v != v ? 0u : v == 0.f ? 0x80000000u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A row as 16-byte pieces at 16-byte addresses: piece j holds tokens [PER j - head, + PER); what lies
// outside the row is not read.
template <bool F32>
struct Row {
  static constexpr int PER = F32 ? 4 : 8, ES = F32 ? 4 : 2;
  const unsigned char* base;  // of token 0
  int V, head;
  __device__ __forceinline__ Row(const LogprobArgs& p, size_t row) {
    base = static_cast<const unsigned char*>(p.x) + (size_t)(row * p.stride) * ES;
    V = p.V;
    head = (int)((uintptr_t)base & 15) / ES;
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (F32) return reinterpret_cast<const float*>(base)[i];
    return dm_bf2f(reinterpret_cast<const bf16_t*>(base)[i]);
  }
  __device__ __forceinline__ int first(int piece) const { return PER * piece - head; }
  __device__ __forceinline__ bool inside(int piece) const { return first(piece) >= 0 && first(piece) + PER <= V; }
  __device__ __forceinline__ u32x4_t raw(int piece) const { return *reinterpret_cast<const u32x4_t*>(base + (ptrdiff_t)ES * first(piece)); }
  static __device__ __forceinline__ void values(const u32x4_t& w, float (&x)[PER]) {
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
  // -inf outside the row
  __device__ __forceinline__ void load(int piece, float (&x)[PER]) const {
    if (inside(piece)) {
      values(raw(piece), x);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int t = first(piece) + i;
        x[i] = t >= 0 && t < V ? at(t) : -DM_INF;
      }
    }
  }
};

// (m, L, S, C) of two parts as one: S follows the reference point, e^(x - m') (x - m') = f (e^(x - m) (x - m) + e^(x - m) (m - m')).
__device__ __forceinline__ void move_to(float m_new, float& m, float& l, float& s, float& c) {
  const float d = __builtin_elementwise_maximum(m - m_new, kFloor), f = dm_exp(d);  // (m = -inf: nothing there yet, or NaN, which stays)
  s = f * dm_fma(l, d, s);
  l *= f;
  c *= f;
  m = m_new;
}

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
  float m = -DM_INF, l = 0.f, s = 0.f, c = 0.f;
  for (int g = w * p.run; g < g_end; ++g) {
    float best = -DM_INF;
    bool low = false;
    for (int st = 0; st < p.steps; st += 2) {
      float x[2][PER];
      const int piece = (g * p.steps + st) * 64 + lane;
      r.load(piece, x[0]);
      r.load(piece + 64, x[1]);
      float mx = -DM_INF;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < PER; ++i) mx = fmaxf(mx, x[u][i]);
      mx = dm_wave_max<64>(mx);
      if (mx == -DM_INF) {  // masked tokens or NaN only: which of them
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            const int t = r.first(piece + 64 * u) + i;
            low = low || (t >= 0 && t < p.V && x[u][i] == -DM_INF);
          }
      }
      best = fmaxf(best, mx);
      if (mx > m) move_to(mx, m, l, s, c);
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
  if (lane == 0) p.sums[row * p.runs + w] = make_float4(m, l, s, c);
}

__device__ __forceinline__ float wg_sum(float v, float* red) {
  v = dm_wave_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[threadIdx.x & 15];
  return dm_row_sum(v);
}
__device__ __forceinline__ float wg_max(float v, float* red) {
  v = dm_wave_max<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return dm_wave_max<16>(red[threadIdx.x & 15]);
}

// grid (rows)
template <bool F32>
__global__ __launch_bounds__(kFinish) void logprobs_finish_kernel(LogprobArgs p) {
  using R = Row<F32>;
  constexpr int PER = R::PER;
  __shared__ float red[16];
  __shared__ uint32_t keys[kGroups];
  __shared__ int chosen[kMaxTop];          // groups, ascending
  __shared__ uint32_t cand_o[kCands];
  __shared__ uint32_t cand_i[kCands];
  __shared__ int n_cands, count[2], fill[17];
  __shared__ uint32_t least;               // order of the k-th best group's best
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.x;
  const R r(p, row);

  if (p.k) {
    for (int g = tid; g < p.groups; g += kFinish) keys[g] = p.best[row * p.groups + g];
    if (tid < kMaxTop) chosen[tid] = 0x7fffffff;
    if (tid == 0) n_cands = 0;
  }
  // the row's sums, and the tokens that were asked for
  float m = -DM_INF, l = 0.f, s = 0.f, c = 0.f;
  float4 part = make_float4(-DM_INF, 0.f, 0.f, 0.f);
  if (tid < p.runs) part = p.sums[row * p.runs + tid];  // (runs <= kGroups <= the workgroup)
  m = wg_max(part.x, red);
  if (part.x < m) move_to(m, part.x, part.y, part.z, part.w);
  l = wg_sum(part.y, red);
  s = wg_sum(part.z, red);
  c = wg_sum(part.w, red);
  const float ref = m > -DM_INF ? m : 0.f;
  l = dm_fma(kLn2, dm_fma(kL2ELow, s, c), l);
  const bool none = l == 0.f;
  const float logl = none ? 0.f : dm_log(l);
  if (tid == 0) {
    if (p.lse) p.lse[row] = none ? -DM_INF : ref + logl;
    if (p.entropy) p.entropy[row] = none ? 0.f : logl - s / l;
  }
  for (int i = tid; i < p.n_tokens; i += kFinish) {
    const uint32_t t = p.tokens[row * p.n_tokens + i];
    p.logprobs[row * p.n_tokens + i] = t < (uint32_t)p.V ? (r.at(t) - ref) - logl : -DM_INF;
  }
  if (p.k == 0) return;

  // the k best groups: a group's rank is how many come before it, counted by 1024 / 512 threads each
  const int kg = min(p.k, p.groups);
  {
    const int g = tid >> 1, part_of = tid & 1;
    int rank = 0;
    const uint32_t mine = g < p.groups ? keys[g] : 0;
    const int half = (p.groups + 1) / 2, lo = part_of * half, hi = min(p.groups, lo + half);
    for (int o = lo; o < hi; ++o) rank += keys[o] > mine || (keys[o] == mine && o < g);
    rank += __shfl_xor(rank, 1, 64);
    __syncthreads();
    if (g < p.groups && part_of == 0 && rank < kg) chosen[rank] = g;
    if (g < p.groups && part_of == 0 && rank == kg - 1) least = mine;
  }
  __syncthreads();
  // in ascending order, so that places in the list go with token ids
  if (tid < 64) {
    const int g = tid < kg ? chosen[tid] : 0x7fffffff;
    int rank = 0;
    for (int o = 0; o < kg; ++o) rank += __builtin_amdgcn_readlane(g, o) < g;
    if (tid < kg) chosen[rank] = g;
  }
  __syncthreads();

  // the tokens of those groups: who is at least as good as the k-th group's best
  const int ppg = 64 * p.steps, pieces = kg * ppg;  // 16-byte pieces
  auto piece_of = [&](int i) { return chosen[i / ppg] * ppg + i % ppg; };
  const uint32_t bound = kg < p.k ? 0 : least;  // (fewer groups than alternatives: all of their tokens)
  // the lanes that have one put it into the list, which has no order: it is ranked by value and id
  auto push = [&](bool has, uint32_t o, int t) {
    const uint64_t mask = __builtin_amdgcn_ballot_w64(has);
    if (mask == 0) return;
    int at = 0;
    if (lane == 0) at = atomicAdd(&n_cands, __popcll(mask));
    at = __builtin_amdgcn_readfirstlane(at) + __popcll(mask & ((uint64_t(1) << lane) - 1));
    if (has && at < kCands) {
      cand_o[at] = o;
      cand_i[at] = t;
    }
  };
  // every token of the chosen groups, in passes of 1024 pieces that all threads go through
  auto look = [&](auto&& f) {
    for (int i0 = 0; i0 < pieces; i0 += kFinish) {
      const int i = i0 + tid;
      float x[PER] = {};
      int t0 = p.V;
      if (i < pieces) {
        const int piece = piece_of(i);
        r.load(piece, x);
        t0 = r.first(piece);
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) f(t0 + e >= 0 && t0 + e < p.V, order_of(x[e]), t0 + e);
    }
  };
  look([&](bool in, uint32_t o, int t) { push(in && o >= bound, o, t); });
  __syncthreads();
  int n = n_cands;
  if (n > kCands) {
    // Many equal tokens, or many good ones in one group: the k-th best value is found bit by bit, then
    // all that are better are taken and, of its equals, those of the lowest ids.
    uint32_t kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t tryit = kth | 1u << bit;
      int have = 0;
      look([&](bool in, uint32_t o, int) { have += in && o >= tryit; });
      if (tid < 2) count[tid] = 0;
      __syncthreads();
      for (int sft = 32; sft; sft >>= 1) have += __shfl_xor(have, sft, 64);
      if (lane == 0) atomicAdd(&count[0], have);
      __syncthreads();
      if (count[0] >= p.k) kth = tryit;
      __syncthreads();
    }
    if (tid == 0) n_cands = 0;
    if (tid == 0) count[1] = 0;
    __syncthreads();
    // the better ones (fewer than k) first: any order
    look([&](bool in, uint32_t o, int t) { push(in && o > kth, o, t); });
    __syncthreads();
    const int better = n_cands;
    // the equals in the order of their ids: passes of 1024 pieces, a prefix sum over the workgroup each
    for (int i0 = 0; i0 < pieces; i0 += kFinish) {
      const int i = i0 + tid;
      uint32_t equal = 0;
      int t0 = 0;
      if (i < pieces) {
        const int piece = piece_of(i);
        float x[PER];
        r.load(piece, x);
        t0 = r.first(piece);
#pragma unroll
        for (int e = 0; e < PER; ++e) equal |= (uint32_t)(order_of(x[e]) == kth && t0 + e >= 0 && t0 + e < p.V) << e;
      }
      const int mine = __popc(equal);
      int before = mine;  // inclusive over the wavefront
      for (int sft = 1; sft < 64; sft <<= 1) {
        const int o = __shfl_up(before, sft, 64);
        if (lane >= sft) before += o;
      }
      if (lane == 63) fill[wave] = before;
      __syncthreads();
      int at = better + count[1] + before - mine;
      for (int wv = 0; wv < wave; ++wv) at += fill[wv];
      for (int e = 0; e < PER; ++e)
        if (equal >> e & 1) {
          if (at < p.k) {
            cand_o[at] = kth;
            cand_i[at] = t0 + e;
          }
          ++at;
        }
      __syncthreads();
      if (tid == 0)
        for (int wv = 0; wv < 16; ++wv) count[1] += fill[wv];
      __syncthreads();
      if (better + count[1] >= p.k) break;
    }
    n = p.k;
  }
  // rank them
  for (int i = tid; i < n; i += kFinish) {
    const uint32_t o = cand_o[i], id = cand_i[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand_o[j] > o || (cand_o[j] == o && cand_i[j] < id);
    if (rank < p.k) {
      p.top_ids[row * p.k + rank] = id;
      p.top_logprobs[row * p.k + rank] = (r.at(id) - ref) - logl;
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
  ORN_REQUIRE(k >= 0 && k <= kMaxTop && k <= V, "token_logprobs: %d alternatives of %d tokens (at most %d)", k, V, kMaxTop);
  ORN_REQUIRE(k == 0 || (d_top_ids && d_top_logprobs), "token_logprobs: alternatives without their arrays");
  ORN_REQUIRE(((uintptr_t)d_logits & (dtype == ORNITH_F32 ? 3 : 1)) == 0, "token_logprobs: misaligned logits");
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
  // groups of 2 KB, longer ones only where a row would have more than kGroups of them
  const int per = dtype == ORNITH_F32 ? 4 : 8;
  const int64_t pieces = ((int64_t)V + 2 * per - 2) / per;  // at any alignment
  p.steps = 2;
  while ((pieces + 64 * p.steps - 1) / (64 * p.steps) > kGroups) p.steps *= 2;
  p.groups = (int)((pieces + 64 * p.steps - 1) / (64 * p.steps));
  // a wavefront takes one group while that fills the machine, eight where there are rows enough
  p.run = (int)std::min<int64_t>(8, std::max<int64_t>(1, (int64_t)rows * p.groups / (32 * ctx->compute_units)));
  p.runs = (p.groups + p.run - 1) / p.run;
  void* base = nullptr;
  if (int rc = ornith_scratch(ctx, (size_t)rows * (p.runs * sizeof(float4) + p.groups * 4) + 512, &base)) return rc;
  ScratchCursor sc(base);
  p.sums = sc.take<float4>((size_t)rows * p.runs);
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
