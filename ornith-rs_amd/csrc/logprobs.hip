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

namespace {

constexpr int kMaxTop = 32;  // alternatives a row

struct LogprobArgs {
  const void* x;
  const uint32_t* tokens;  // [rows, n_tokens]
  float* logprobs;         // [rows, n_tokens]
  float* entropy;          // [rows]
  float* lse;              // [rows]
  uint32_t* top_ids;       // [rows, k]
  float* top_logprobs;     // [rows, k]
  int64_t stride;
  int V, n_tokens, k;
};

template <bool F32>
__device__ __forceinline__ float logit(const LogprobArgs& p, size_t row, int i) {
  if constexpr (F32) return static_cast<const float*>(p.x)[row * p.stride + i];
  return dm_bf2f(static_cast<const bf16_t*>(p.x)[row * p.stride + i]);
}

// A logit and its index as one number, larger for a larger value and, among equal values, for a
// lower index; NaN below everything.
__device__ __forceinline__ uint64_t order_key(float v, uint32_t i) {
  uint32_t u = __float_as_uint(v);
  u = v != v ? 0u : v == 0.f ? 0x80000000u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)~i;
}

// One workgroup a row.
template <bool F32>
__global__ __launch_bounds__(1024) void logprobs_kernel(LogprobArgs p) {
  __shared__ float red[3][16];
  __shared__ uint64_t best[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.x;
  float m = -DM_INF;
  for (int i = tid; i < p.V; i += 1024) m = fmaxf(m, logit<F32>(p, row, i));
  m = dm_wave_max<64>(m);
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  for (int w = 0; w < 16; ++w) m = fmaxf(m, red[0][w]);
  const float ref = m > -DM_INF ? m : 0.f;  // (a row with nothing but masked tokens)
  float l = 0.f, s = 0.f;
  for (int i = tid; i < p.V; i += 1024) {
    const float d = logit<F32>(p, row, i) - ref, e = __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
    l += e;
    s += e != 0.f ? e * d : 0.f;
  }
  l = dm_wave_sum<64>(l);
  s = dm_wave_sum<64>(s);
  if (lane == 0) {
    red[1][wave] = l;
    red[2][wave] = s;
  }
  __syncthreads();
  l = s = 0.f;
  for (int w = 0; w < 16; ++w) {
    l += red[1][w];
    s += red[2][w];
  }
  const bool none = l == 0.f;
  const float logl = none ? 0.f : dm_log(l);
  if (tid == 0) {
    if (p.lse) p.lse[row] = none ? -DM_INF : ref + logl;
    if (p.entropy) p.entropy[row] = none ? 0.f : logl - s / l;
  }
  for (int i = tid; i < p.n_tokens; i += 1024) {
    const uint32_t t = p.tokens[row * p.n_tokens + i];
    p.logprobs[row * p.n_tokens + i] = t < (uint32_t)p.V ? (logit<F32>(p, row, t) - ref) - logl : -DM_INF;
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < p.k; ++j) {
    uint64_t b = 0;
    for (int i = tid; i < p.V; i += 1024) {
      const uint64_t key = order_key(logit<F32>(p, row, i), i);
      if (key < last && key > b) b = key;
    }
    for (int sft = 32; sft; sft >>= 1) {
      const uint64_t o = __shfl_xor(b, sft, 64);
      b = o > b ? o : b;
    }
    __syncthreads();
    if (lane == 0) best[wave] = b;
    __syncthreads();
    for (int w = 0; w < 16; ++w) b = best[w] > b ? best[w] : b;
    last = b;
    if (tid == 0) {
      const uint32_t id = ~(uint32_t)b;
      p.top_ids[row * p.k + j] = id;
      p.top_logprobs[row * p.k + j] = (logit<F32>(p, row, id) - ref) - logl;
    }
  }
}

}  // namespace

extern "C" int ornith_token_logprobs(ornith_ctx* ctx, const void* d_logits, int dtype, int rows, int V, int64_t row_stride,
                                     const uint32_t* d_tokens, int n_tokens, int k, float* d_logprobs, float* d_entropy,
                                     float* d_lse, uint32_t* d_top_ids, float* d_top_logprobs) {
  ORN_REQUIRE(d_logits, "token_logprobs: null logits");
  ORN_REQUIRE(dtype == ORNITH_F32 || dtype == ORNITH_BF16, "token_logprobs: dtype %d", dtype);
  ORN_REQUIRE(rows >= 1 && V >= 1 && row_stride >= V, "token_logprobs: rows=%d V=%d row_stride=%lld", rows, V, (long long)row_stride);
  ORN_REQUIRE(n_tokens >= 0 && (n_tokens == 0 || (d_tokens && d_logprobs)), "token_logprobs: %d tokens a row without their arrays", n_tokens);
  ORN_REQUIRE(k >= 0 && k <= kMaxTop && k <= V, "token_logprobs: %d alternatives of %d tokens (at most %d)", k, V, kMaxTop);
  ORN_REQUIRE(k == 0 || (d_top_ids && d_top_logprobs), "token_logprobs: alternatives without their arrays");
  ORN_REQUIRE(((uintptr_t)d_logits & (dtype == ORNITH_F32 ? 3 : 1)) == 0, "token_logprobs: misaligned logits");
  ORN_REQUIRE(ctx, "token_logprobs: null context");
  const OrnDevice on(ctx);
  const LogprobArgs p{d_logits, d_tokens, d_logprobs, d_entropy, d_lse, d_top_ids, d_top_logprobs, row_stride, V, n_tokens, k};
  if (dtype == ORNITH_F32)
    hipLaunchKernelGGL(logprobs_kernel<true>, dim3(rows), dim3(1024), 0, ctx->stream, p);
  else
    hipLaunchKernelGGL(logprobs_kernel<false>, dim3(rows), dim3(1024), 0, ctx->stream, p);
  ORN_LAUNCH_CHECK("logprobs_kernel");
  return ORNITH_OK;
}
