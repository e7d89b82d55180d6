// kv4.cu -- writing and reading the 4-bit kv cache (format: kv4.cuh).
//
// kv4_append_kernel: k and v rows of new tokens (bf16 or fp32, any token / head strides) -> codes and
// params at (slots[t], positions[t]) of the pool.  Eight lanes hold a group's 64 features (8 each, one
// or two 16-byte loads), find its minimum and maximum with three shuffles and write one 32-bit word of
// codes each: 32 contiguous bytes per group.  Each input byte is read once, 36 bytes per group are written;
// bound for long prompts: the instructions (about 15 a feature) before HBM, and latency for a decode step.
// kv4_read_kernel: the fp32 / bf16 values of given rows, four features a lane.
// Append and read of 8190 x 4 rows of 128 (fp32): 23 us together, 3.1 TB/s; of 64 tokens 3.7 us
// (four groups a thread of the read kernel: 22.5 and 5.1).
#include "kv4.cuh"

namespace ccut {

template <bool BF16>
CCUT_DEVICE void load8(const void* base, long long off, float (&x)[8]) {
  if constexpr (BF16) {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + off);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + off);
    const float4 a = p[0], b = p[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
}

struct Kv4In {
  const void* x;
  long long token_stride, head_stride;  // elements
  uint8_t* codes;
  __half2* params;
};

CCUT_DEVICE float kv4_max3(float a, float b, float c) {  // NaN when one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
CCUT_DEVICE float kv4_min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A code before the clamp to 0..15 is rint(fl32(d / s)).  d (1 / s) is within 2^-17 of that quotient where the clamp
// leaves anything, so where it is further than 2^-15 from the middle of two integers it rounds to the same one;
// the rest take the division (for every code it took 19 us of 8190 x 4 fp32 rows of 128, cold, where this takes 14).
CCUT_DEVICE uint32_t kv4_codes(const float (&x)[8], float m, float s) {
  const float r = __frcp_rn(s), magic = 12582912.f;  // 1.5 2^23: y + magic has the rounded y in its low bits
  const u64 m2 = pf_pair(-m, -m), r2 = pf_pair(r, r), up = pf_pair(magic, magic), down = pf_pair(-magic, -magic);
  uint32_t w = 0;
  float worst = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float y0, y1, u0, u1, d0, d1;
    pf_unpair(pf_mul2(pf_add2(pf_pair(x[i], x[i + 1]), m2), r2), y0, y1);
    const u64 y = pf_pair(fminf(fmaxf(y0, 0.f), 15.f), fminf(fmaxf(y1, 0.f), 15.f)), u = pf_add2(y, up);
    pf_unpair(u, u0, u1);
    pf_unpair(pf_fma2(pf_add2(u, down), pf_pair(-1.f, -1.f), y), d0, d1);  // y - its integer, exact
    worst = pf_max3(worst, fabsf(d0), fabsf(d1));
    w += (__float_as_uint(u0) << (4 * i)) + (__float_as_uint(u1) << (4 * i + 4));
  }
  w -= 0x4B400000u * 0x11111111u;  // the exponents
  if (worst > 0.5f - 0x1p-15f) {
    w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[i], m), s)), 0.f), 15.f) << (4 * i);
  }
  return w;
}

// blockIdx.y: 0 = k, 1 = v.  Eight consecutive lanes per (token, head, group).
template <bool K_BF16, bool V_BF16>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4In k, Kv4In v, int tokens, int kv_heads, int groups,
                                                         const int32_t* __restrict__ slots,
                                                         const int32_t* __restrict__ positions, int max_len,
                                                         long long slot_rows, int num_slots) {
  pdl_wait();
  pdl_trigger();
  const unsigned item = blockIdx.x * 32 + (threadIdx.x >> 3);
  const int lane8 = threadIdx.x & 7;
  const unsigned per_token = kv_heads * groups;
  const unsigned t = item / per_token, hg = item - t * per_token;
  if (t >= (unsigned)tokens) return;
  const int h = hg / groups, g = hg % groups;
  const int slot = slots[t], pos = positions[t];
  const bool store = slot >= 0 && slot < num_slots && pos >= 0 && pos < max_len;
  const unsigned mask = 0xFFu << (threadIdx.x & 24);  // the item's eight lanes
  const Kv4In in = blockIdx.y ? v : k;
  float x[8];
  const long long off = t * in.token_stride + h * in.head_stride + g * kKv4Group + lane8 * 8;
  if (blockIdx.y) load8<V_BF16>(in.x, off, x);
  else load8<K_BF16>(in.x, off, x);
  // the least and the largest, NaN if one is there
  float lo = kv4_min3(kv4_min3(x[0], x[1], x[2]), kv4_min3(x[3], x[4], x[5]), fminf(x[6], x[7]));
  float hi = kv4_max3(kv4_max3(x[0], x[1], x[2]), kv4_max3(x[3], x[4], x[5]), kv4_max3(x[6], x[7], x[7]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    const float h = __shfl_xor_sync(mask, hi, o);
    lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
    hi = kv4_max3(hi, h, h);
  }
  const bool bad = !(hi <= 3.402823466e38f && lo >= -3.402823466e38f);
  lo = fminf(fmaxf(lo, -65504.f), 65504.f);
  hi = fminf(fmaxf(hi, -65504.f), 65504.f);
  __half m = __float2half_rn(lo);
  const float mf = __half2float(m);
  __half s = __float2half_rn(fmaxf(__fmul_rn(__fsub_rn(hi, mf), 0.06666667f), 0.f));
  const float sf = __half2float(s);
  const uint32_t w = sf > 0.f && !bad ? kv4_codes(x, mf, sf) : 0;
  if (bad) s = m = __ushort_as_half(0x7FFF);
  if (!store) return;
  const size_t row = (size_t)slot * (size_t)slot_rows + (size_t)h * max_len + pos;
  *reinterpret_cast<uint32_t*>(in.codes + (row * groups + g) * (kKv4Group / 2) + lane8 * 4) = w;
  if (lane8 == 0) in.params[row * groups + g] = __halves2half2(s, m);
}

// Values of rows (slots[t], positions[t]): out [tokens, kv_heads, d]; rows outside the pool read zero.
template <bool OUT_BF16>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* __restrict__ kc, const __half2* __restrict__ kp,
                                                       const uint8_t* __restrict__ vc, const __half2* __restrict__ vp,
                                                       const int32_t* __restrict__ slots,
                                                       const int32_t* __restrict__ positions, int tokens, int kv_heads,
                                                       int groups, int max_len, long long slot_rows, int num_slots,
                                                       void* __restrict__ k_out, void* __restrict__ v_out) {
  pdl_wait();
  pdl_trigger();
  // a group of a row, four features a lane: every store instruction of a warp writes whole lines
  const unsigned item = blockIdx.x * 16 + (threadIdx.x >> 4);
  const int lane16 = threadIdx.x & 15;
  const unsigned per_token = kv_heads * groups;
  const unsigned t = item / per_token, hg = item - t * per_token;
  if (t >= (unsigned)tokens) return;
  const int h = hg / groups, g = hg % groups;
  const int slot = slots[t], pos = positions[t];
  uint32_t w = 0;
  float2 sm = make_float2(0.f, 0.f);
  if (slot >= 0 && slot < num_slots && pos >= 0 && pos < max_len) {
    const size_t at = ((size_t)slot * (size_t)slot_rows + (size_t)h * max_len + pos) * groups + g;
    w = reinterpret_cast<const uint16_t*>(blockIdx.y ? vc : kc)[at * 16 + lane16];
    sm = __half22float2((blockIdx.y ? vp : kp)[at]);
  }
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = kv4_value((w >> (4 * i)) & 15, sm.x, sm.y);
  const size_t idx = (size_t)item * 16 + lane16;
  void* out = blockIdx.y ? v_out : k_out;
  if constexpr (OUT_BF16) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(x[0], x[1]), hi = __floats2bfloat162_rn(x[2], x[3]);
    reinterpret_cast<uint2*>(out)[idx] =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  } else {
    reinterpret_cast<float4*>(out)[idx] = make_float4(x[0], x[1], x[2], x[3]);
  }
}

static bool float_dtype(int t) { return t == CCUT_OUT_BF16 || t == CCUT_OUT_F32; }

}  // namespace ccut

using namespace ccut;

extern "C" {

int ccut_kv4_append(const void* k, int k_dtype, long long k_token_stride, long long k_head_stride, const void* v,
                    int v_dtype, long long v_token_stride, long long v_head_stride, int tokens, int kv_heads,
                    int head_dim, const int32_t* slots, const int32_t* positions, uint8_t* k_codes,
                    uint16_t* k_params, uint8_t* v_codes, uint16_t* v_params, int max_len, long long slot_rows,
                    int num_slots, ccut_stream_t stream) {
  PdlScope pdl_scope(tokens);
  if (head_dim != 64 && head_dim != 128) return CCUT_ERR_UNSUPPORTED;
  if (tokens < 0 || !kv4_shape_ok(kv_heads, head_dim, max_len, slot_rows, num_slots)) return CCUT_ERR_INVALID;
  if (!float_dtype(k_dtype) || !float_dtype(v_dtype)) return CCUT_ERR_INVALID;
  if (tokens == 0) return CCUT_OK;
  if (!k || !v || !slots || !positions || (num_slots > 0 && (!k_codes || !k_params || !v_codes || !v_params)))
    return CCUT_ERR_INVALID;
  if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) % 8) return CCUT_ERR_INVALID;
  if (misaligned(k, 16) || misaligned(v, 16) || misaligned(k_codes, 16) || misaligned(v_codes, 16) ||
      misaligned(k_params, head_dim / 16) || misaligned(v_params, head_dim / 16))
    return CCUT_ERR_INVALID;
  const int groups = head_dim / kKv4Group;
  const long long blocks = ((long long)tokens * kv_heads * groups + 31) / 32;
  if (blocks > 2147483647LL / 32) return CCUT_ERR_UNSUPPORTED;  // items in 31 bits: 274 GB of bf16 rows and more
  const Kv4In ki{k, k_token_stride, k_head_stride, k_codes, reinterpret_cast<__half2*>(k_params)};
  const Kv4In vi{v, v_token_stride, v_head_stride, v_codes, reinterpret_cast<__half2*>(v_params)};
  const bool kb = k_dtype == CCUT_OUT_BF16, vb = v_dtype == CCUT_OUT_BF16;
  auto kern = kb ? (vb ? kv4_append_kernel<true, true> : kv4_append_kernel<true, false>)
                 : (vb ? kv4_append_kernel<false, true> : kv4_append_kernel<false, false>);
  return launch_k(kern, dim3((unsigned)blocks, 2), dim3(256), 0, stream, ki, vi, tokens, kv_heads, groups, slots,
                  positions, max_len, slot_rows, num_slots);
}

int ccut_kv4_read(const uint8_t* k_codes, const uint16_t* k_params, const uint8_t* v_codes, const uint16_t* v_params,
                  const int32_t* slots, const int32_t* positions, int tokens, int kv_heads, int head_dim, int max_len,
                  long long slot_rows, int num_slots, void* k_out, void* v_out, int out_dtype, ccut_stream_t stream) {
  PdlScope pdl_scope(tokens);
  if (head_dim != 64 && head_dim != 128) return CCUT_ERR_UNSUPPORTED;
  if (tokens < 0 || !kv4_shape_ok(kv_heads, head_dim, max_len, slot_rows, num_slots) || !float_dtype(out_dtype))
    return CCUT_ERR_INVALID;
  if (tokens == 0) return CCUT_OK;
  if (!k_out || !v_out || !slots || !positions || (num_slots > 0 && (!k_codes || !k_params || !v_codes || !v_params)))
    return CCUT_ERR_INVALID;
  if (misaligned(k_out, 16) || misaligned(v_out, 16) || misaligned(k_codes, 16) || misaligned(v_codes, 16) ||
      misaligned(k_params, head_dim / 16) || misaligned(v_params, head_dim / 16))
    return CCUT_ERR_INVALID;
  const int groups = head_dim / kKv4Group;
  const long long blocks = ((long long)tokens * kv_heads * groups + 15) / 16;
  if (blocks > 2147483647LL / 16) return CCUT_ERR_UNSUPPORTED;  // items in 31 bits: 274 GB of bf16 rows and more
  auto kern = out_dtype == CCUT_OUT_BF16 ? kv4_read_kernel<true> : kv4_read_kernel<false>;
  return launch_k(kern, dim3((unsigned)blocks, 2), dim3(256), 0, stream, k_codes,
                  reinterpret_cast<const __half2*>(k_params), v_codes, reinterpret_cast<const __half2*>(v_params),
                  slots, positions, tokens, kv_heads, groups, max_len, slot_rows, num_slots, k_out, v_out);
}

}  // extern "C"
