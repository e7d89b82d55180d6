// kv4_attn.cu -- grouped-query attention over the 4-bit kv cache (format: kv4.cuh).
//
// q bf16 [batch, heads, seq, d]; batch row b reads slot slots[b], its query i sees positions
// <= starts[b] + i (and < kv_len); query head h reads kv head h / (heads / kv_heads).
//   x_j = scale * sum_d q_d (s_jg c_jd + m_jg), optionally soft-capped; o = sum_j softmax(x)_j v^_j
#include <math.h>

#include "kv4.cuh"

namespace ccut {

constexpr int kKv4Chunk = 256;  // positions per split

struct Kv4AttnArgs {
  const uint16_t* q;
  const uint8_t* kc;
  const __half2* kp;
  const uint8_t* vc;
  const __half2* vp;
  const int32_t* slots;
  const int32_t* starts;
  int heads, kv_heads, seq, max_len, kv_len, num_slots;
  long long slot_rows;
  float scale, softcap;
  void* out;
  float* part;
};

// One CTA per (query row, split of 256 positions): thread j scores positions j and j + 128, then
// thread d accumulates feature d.
template <int D, bool OUT_BF16>
__global__ void __launch_bounds__(128) kv4_attn_simple_kernel(Kv4AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int G = D / kKv4Group;
  __shared__ float qs[D], p[kKv4Chunk], red[8];
  const int tid = threadIdx.x;
  const long long row = blockIdx.x;  // (b * heads + h) * seq + i
  const int i = (int)(row % a.seq), h = (int)(row / a.seq % a.heads), b = (int)(row / a.seq / a.heads);
  const int slot = a.slots[b], start = a.starts[b];
  int n = min(a.kv_len, min(start, a.kv_len) + i + 1);
  if (slot < 0 || slot >= a.num_slots || start < 0) n = 0;
  const int p0 = blockIdx.y * kKv4Chunk, p1 = min(n, p0 + kKv4Chunk);
  const size_t r0 = n > 0 ? (size_t)slot * (size_t)a.slot_rows + (size_t)(h / (a.heads / a.kv_heads)) * a.max_len : 0;
  if (tid < D) qs[tid] = __uint_as_float((uint32_t)a.q[row * D + tid] << 16);
  __syncthreads();
  float mx = -INFINITY;
  for (int j = p0 + tid; j < p1; j += 128) {
    const uint32_t* c = reinterpret_cast<const uint32_t*>(a.kc) + (r0 + j) * (D / 8);
    float x = 0.f;
    for (int w = 0; w < D / 8; ++w) {
      const float2 sm = __half22float2(a.kp[(r0 + j) * G + w / 8]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x = fmaf(qs[w * 8 + e], kv4_value((c[w] >> (4 * e)) & 15, sm.x, sm.y), x);
    }
    x *= a.scale;
    if (a.softcap > 0.f) x = tanhf(x / a.softcap) * a.softcap;
    p[j - p0] = x;
    mx = fmaxf(mx, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if ((tid & 31) == 0) red[tid >> 5] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float l = 0.f;
  for (int j = p0 + tid; j < p1; j += 128) {
    const float e = expf(p[j - p0] - mx);
    p[j - p0] = e;
    l += e;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  if ((tid & 31) == 0) red[4 + (tid >> 5)] = l;
  __syncthreads();
  l = (red[4] + red[5]) + (red[6] + red[7]);
  float o = 0.f;
  if (tid < D) {
    for (int j = p0; j < p1; ++j) {
      const uint32_t q = a.vc[(r0 + j) * (D / 2) + tid / 2] >> (4 * (tid & 1));
      const float2 sm = __half22float2(a.vp[(r0 + j) * G + tid / kKv4Group]);
      o = fmaf(p[j - p0], kv4_value(q & 15, sm.x, sm.y), o);
    }
    if (gridDim.y > 1) {
      float* w = a.part + ((size_t)blockIdx.y * gridDim.x + row) * (D + 2);
      w[2 + tid] = o;
      if (tid == 0) w[0] = mx, w[1] = l;
    } else {
      o = l > 0.f ? o / l : (l == 0.f ? 0.f : o / l);
      if constexpr (OUT_BF16) static_cast<__nv_bfloat16*>(a.out)[row * D + tid] = __float2bfloat16_rn(o);
      else static_cast<float*>(a.out)[row * D + tid] = o;
    }
  }
}

// Merge of the splits: one warp per query row, in split order.
template <int D, bool OUT_BF16>
__global__ void __launch_bounds__(256) kv4_merge_kernel(const float* __restrict__ part, long long rows, int splits,
                                                        void* __restrict__ out) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = D / 32;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float M = -INFINITY, L = 0.f, o[E] = {};
  bool nan = false;
  for (int s = 0; s < splits; ++s) {
    const float* w = part + ((size_t)s * rows + row) * (D + 2);
    M = fmaxf(M, w[0]);
    nan |= isnan(w[1]);
  }
  for (int s = 0; s < splits; ++s) {
    const float* w = part + ((size_t)s * rows + row) * (D + 2);
    if (w[0] == -INFINITY && !isnan(w[1])) continue;  // a split that saw nothing
    const float f = expf(w[0] - M);
    L = fmaf(w[1], f, L);
#pragma unroll
    for (int j = 0; j < E; ++j) o[j] = fmaf(w[2 + lane + 32 * j], f, o[j]);
  }
  if (nan) L = __int_as_float(0x7FFFFFFF);
#pragma unroll
  for (int j = 0; j < E; ++j) {
    const float v = L == 0.f ? 0.f : o[j] / L;
    if constexpr (OUT_BF16) static_cast<__nv_bfloat16*>(out)[row * D + lane + 32 * j] = __float2bfloat16_rn(v);
    else static_cast<float*>(out)[row * D + lane + 32 * j] = v;
  }
}

static int kv4_splits(int kv_len) { return kv_len > 0 ? (kv_len + kKv4Chunk - 1) / kKv4Chunk : 1; }

template <int D>
static int run_kv4_attention(const Kv4AttnArgs& a, long long rows, bool ob, cudaStream_t st) {
  const int sp = kv4_splits(a.kv_len);
  auto kern = ob ? kv4_attn_simple_kernel<D, true> : kv4_attn_simple_kernel<D, false>;
  int rc = launch_k(kern, dim3((unsigned)rows, sp), dim3(128), 0, st, a);
  if (rc || sp == 1) return rc;
  auto merge = ob ? kv4_merge_kernel<D, true> : kv4_merge_kernel<D, false>;
  return launch_k(merge, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, (const float*)a.part, rows, sp, a.out);
}

}  // namespace ccut

using namespace ccut;

extern "C" {

size_t ccut_kv4_attention_workspace_bytes(int batch, int heads, int kv_heads, int seq, int kv_len, int head_dim) {
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq < 0 || kv_len < 0 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  const int sp = kv4_splits(kv_len);
  if (sp <= 1) return 256;
  return 256 + (size_t)sp * batch * heads * seq * (head_dim + 2) * sizeof(float);
}

int ccut_kv4_attention(const uint16_t* q, const uint8_t* k_codes, const uint16_t* k_params, const uint8_t* v_codes,
                       const uint16_t* v_params, const int32_t* slots, const int32_t* starts, int batch, int heads,
                       int kv_heads, int seq, int head_dim, int max_len, int kv_len, long long slot_rows,
                       int num_slots, float scale, float softcap, void* out, int out_dtype, void* workspace,
                       size_t ws_bytes, ccut_stream_t stream) {
  PdlScope pdl_scope((long)batch * seq);
  if (head_dim != 64 && head_dim != 128) return CCUT_ERR_UNSUPPORTED;
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq < 0 || kv_len < 0 || kv_len > max_len ||
      !kv4_shape_ok(kv_heads, head_dim, max_len, slot_rows, num_slots))
    return CCUT_ERR_INVALID;
  if (out_dtype != CCUT_OUT_BF16 && out_dtype != CCUT_OUT_F32) return CCUT_ERR_INVALID;
  if (batch == 0 || seq == 0) return CCUT_OK;
  if (!q || !out || !slots || !starts || (num_slots > 0 && (!k_codes || !k_params || !v_codes || !v_params)))
    return CCUT_ERR_INVALID;
  if (misaligned(q, 16) || misaligned(k_codes, 16) || misaligned(v_codes, 16) || misaligned(k_params, head_dim / 16) ||
      misaligned(v_params, head_dim / 16) || misaligned(out, 16) || misaligned(workspace, 16))
    return CCUT_ERR_INVALID;
  const long long rows = (long long)batch * heads * seq;
  if (rows > 2147483647LL || kv4_splits(kv_len) > 65535) return CCUT_ERR_UNSUPPORTED;
  if (kv4_splits(kv_len) > 1 &&
      (!workspace || ws_bytes < ccut_kv4_attention_workspace_bytes(batch, heads, kv_heads, seq, kv_len, head_dim)))
    return CCUT_ERR_WORKSPACE;
  if (!(scale > 0.f)) scale = 1.f / sqrtf((float)head_dim);
  Kv4AttnArgs a{q, k_codes, reinterpret_cast<const __half2*>(k_params), v_codes,
                reinterpret_cast<const __half2*>(v_params), slots, starts, heads, kv_heads, seq, max_len, kv_len,
                num_slots, slot_rows, scale, softcap, out,
                workspace ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256) : nullptr};
  const bool ob = out_dtype == CCUT_OUT_BF16;
  return head_dim == 128 ? run_kv4_attention<128>(a, rows, ob, stream) : run_kv4_attention<64>(a, rows, ob, stream);
}

}  // extern "C"
