// logprobs.cu -- log probability, entropy and rank of given tokens, and the top alternatives.
//
// Per row x of vocab logits and its token t, in fp32 (natural logarithms):
//   logZ = m + log sum_v e^(x_v - m), m = max x;  logprob = x_t - logZ;
//   entropy = log sum_v e^(x_v - m) - (sum_v e^(x_v - m) (x_v - m)) / sum_v e^(x_v - m);
//   rank = 1 + #{v: x_v > x_t} + #{v < t: x_v = x_t};
//   top n by descending value, ties to the lowest index, with their log probabilities.
#include <math.h>

#include "host.cuh"

namespace ccut {

template <bool BF16>
CCUT_DEVICE float logit(const void* x, size_t i) {
  if constexpr (BF16) return __uint_as_float((uint32_t) static_cast<const uint16_t*>(x)[i] << 16);
  else return static_cast<const float*>(x)[i];
}

// The order of logits as integers: descending value is descending key, -0 equals +0, NaN comes last.
CCUT_DEVICE int order_key(float x) {
  if (isnan(x)) return -0x7FFFFFFF - 1;
  const int b = __float_as_int(x + 0.f);
  return b < 0 ? b ^ 0x7FFFFFFF : b;
}

CCUT_DEVICE float block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < (int)blockDim.x / 32; ++w) v = fmaxf(v, red[w]);
  return v;
}
CCUT_DEVICE float block_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < (int)blockDim.x / 32; ++w) v += red[w];
  return v;
}

// One CTA per row: a pass for the maximum, one for the sums and the rank, one per alternative.
template <bool BF16>
__global__ void __launch_bounds__(256) logprobs_simple_kernel(const void* __restrict__ logits, int vocab, long long ld,
                                                              const int32_t* __restrict__ tokens, int top_n,
                                                              float* __restrict__ logprob, float* __restrict__ entropy,
                                                              int32_t* __restrict__ rank, int32_t* __restrict__ top_ids,
                                                              float* __restrict__ top_lp) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red[8];
  __shared__ int redi[8], redk[8];
  const size_t base = (size_t)blockIdx.x * (size_t)ld;
  const int t = tokens[blockIdx.x];
  const bool ok = t >= 0 && t < vocab;
  const float xt = ok ? logit<BF16>(logits, base + t) : 0.f;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < vocab; i += 256) m = fmaxf(m, logit<BF16>(logits, base + i));
  m = block_max(m, red);
  float s = 0.f, w = 0.f;
  int r = 0;
  const int kt = order_key(xt);
  for (int i = threadIdx.x; i < vocab; i += 256) {
    const float x = logit<BF16>(logits, base + i), e = expf(x - m);
    s += e;
    if (e > 0.f) w = fmaf(e, x - m, w);
    const int k = order_key(x);
    r += k > kt || (k == kt && i < t);
  }
  s = block_sum(s, red);
  w = block_sum(w, red);
  r = __reduce_add_sync(0xffffffffu, r);
  if ((threadIdx.x & 31) == 0) redi[threadIdx.x >> 5] = r;
  __syncthreads();
  r = 0;
  for (int o = 0; o < 8; ++o) r += redi[o];
  __syncthreads();
  const float lz = logf(s);
  if (threadIdx.x == 0) {
    logprob[blockIdx.x] = ok ? (xt - m) - lz : __int_as_float(0x7FFFFFFF);
    entropy[blockIdx.x] = lz - w / s;
    rank[blockIdx.x] = ok ? 1 + r : 0;
  }
  int lastk = 0x7FFFFFFF, lasti = -1;
  for (int j = 0; j < top_n; ++j) {  // the first entry after (lastk, lasti) in the order
    int bk = -0x7FFFFFFF - 1, bi = 0x7FFFFFFF;
    for (int i = threadIdx.x; i < vocab; i += 256) {
      const int k = order_key(logit<BF16>(logits, base + i));
      if (!(k < lastk || (k == lastk && i > lasti))) continue;
      if (k > bk || (k == bk && i < bi)) bk = k, bi = i;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const int ok2 = __shfl_xor_sync(0xffffffffu, bk, o), oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (ok2 > bk || (ok2 == bk && oi < bi)) bk = ok2, bi = oi;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) redk[threadIdx.x >> 5] = bk, redi[threadIdx.x >> 5] = bi;
    __syncthreads();
    for (int o = 0; o < 8; ++o)
      if (redk[o] > bk || (redk[o] == bk && redi[o] < bi)) bk = redk[o], bi = redi[o];
    lastk = bk;
    lasti = bi;
    if (threadIdx.x == 0) {
      top_ids[(size_t)blockIdx.x * top_n + j] = bi;
      top_lp[(size_t)blockIdx.x * top_n + j] = (logit<BF16>(logits, base + bi) - m) - lz;
    }
  }
}

}  // namespace ccut

using namespace ccut;

extern "C" {

size_t ccut_token_logprobs_workspace_bytes(int rows, int vocab, int top_n) {
  if (rows < 0 || vocab <= 0 || top_n < 0) return 0;
  return 256;
}

int ccut_token_logprobs(const void* logits, int dtype, int rows, int vocab, long long ld, const int32_t* tokens,
                        int top_n, float* logprob, float* entropy, int32_t* rank, int32_t* top_ids,
                        float* top_logprobs, void* workspace, size_t ws_bytes, ccut_stream_t stream) {
  PdlScope pdl_scope(rows);
  if (dtype != CCUT_OUT_BF16 && dtype != CCUT_OUT_F32) return CCUT_ERR_INVALID;
  if (rows < 0 || vocab <= 0 || ld < vocab || top_n < 0 || top_n > vocab) return CCUT_ERR_INVALID;
  if (top_n > CCUT_MAX_TOP_LOGPROBS) return CCUT_ERR_UNSUPPORTED;
  if (rows == 0) return CCUT_OK;
  if (!logits || !tokens || !logprob || !entropy || !rank || (top_n > 0 && (!top_ids || !top_logprobs)))
    return CCUT_ERR_INVALID;
  if (ws_bytes < ccut_token_logprobs_workspace_bytes(rows, vocab, top_n) || !workspace) return CCUT_ERR_WORKSPACE;
  auto kern = dtype == CCUT_OUT_BF16 ? logprobs_simple_kernel<true> : logprobs_simple_kernel<false>;
  return launch_k(kern, dim3(rows), dim3(256), 0, stream, logits, vocab, ld, tokens, top_n, logprob, entropy, rank,
                  top_ids, top_logprobs);
}

}  // extern "C"
