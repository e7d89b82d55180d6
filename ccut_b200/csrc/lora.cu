// lora.cu -- low-rank adapters of many requests beside a shared projection.
//
//   out[t, o] = base[t, o] + scale[a] * sum_r B[a, o, r] * (sum_i A[a, j(o) rank + r, i] x[t, i]),  a = ids[t],
// where j(o) is the slice (q, k or v of a fused projection, say) that output o belongs to; a row whose
// id is outside [0, adapters) keeps its base.
//
// Two launches.  lora_shrink_kernel: partial products h[split, t, slices * rank] of the rows with their
// adapters' A, split over the inputs.  lora_expand_kernel: h summed in split order, scaled, times B,
// added to the base.  Both work on tiles of 16 tokens, the M of m16n8k16 bf16 MMAs, and loop over the
// distinct adapters of the tile; a row takes the result of its own adapter by selection, so nothing of
// another request's adapter (a NaN weight, say) reaches it.
#include "host.cuh"

namespace ccut {

constexpr int kLoraTile = 16;   // tokens per tile
constexpr int kLoraWarps = 4;
constexpr int kLoraMaxRanks = 256;  // slices * rank

struct LoraArgs {
  const uint16_t* x;
  const uint16_t* a;
  const uint16_t* b;
  const float* scales;
  const int32_t* ids;
  int tokens, inputs, outputs, rank, slices, adapters;
  int ends[CCUT_LORA_MAX_SLICES];  // first output past each slice
  const void* base;
  long long base_ld;
  void* out;
  long long out_ld;
  float* part;
  int splits, k_per_split;
};

// The tile's adapter ids (-1 outside [0, adapters) or past the last token) and its distinct adapters in
// order of first appearance; returns their number.
CCUT_DEVICE int tile_adapters(const LoraArgs& p, int t0, int (&ids)[kLoraTile], int (&uniq)[kLoraTile], int& n) {
  if (threadIdx.x < kLoraTile) {
    const int t = t0 + threadIdx.x;
    const int id = t < p.tokens ? p.ids[t] : -1;
    ids[threadIdx.x] = id >= 0 && id < p.adapters ? id : -1;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    for (int i = 0; i < kLoraTile; ++i) {
      bool seen = ids[i] < 0;
      for (int j = 0; j < n; ++j) seen |= uniq[j] == ids[i];
      if (!seen) uniq[n++] = ids[i];
    }
  }
  __syncthreads();
  return n;
}

// Grid (tiles, splits, blocks of 32 rank rows): warp w takes the 8 rows 32 z + 8 w .. of slices * rank.
__global__ void __launch_bounds__(kLoraWarps * 32) lora_shrink_kernel(LoraArgs p) {
  pdl_wait();
  pdl_trigger();
  __shared__ int ids[kLoraTile], uniq[kLoraTile], cnt;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int t0 = blockIdx.x * kLoraTile;
  const int n = tile_adapters(p, t0, ids, uniq, cnt);
  const int R = p.slices * p.rank, r0 = blockIdx.z * 32 + warp * 8;
  if (r0 >= R) return;
  const int k0 = blockIdx.y * p.k_per_split, k1 = min(p.inputs, k0 + p.k_per_split);
  const int row0 = t0 + g, row1 = t0 + g + 8;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  float keep[4] = {0.f, 0.f, 0.f, 0.f};
  for (int u = 0; u < n; ++u) {
    const int a = uniq[u];
    const uint16_t* ar = p.a + ((size_t)a * R + r0 + g) * p.inputs;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    // 32 inputs a step: lane t holds inputs k + 8 t .. + 7 of its rows (the order of the k index of an MMA is free)
    for (int k = k0; k < k1; k += 32) {
      const int kk = k + 8 * t;
      const bool in = kk < k1;
      const uint4 x0 = in && row0 < p.tokens ? *reinterpret_cast<const uint4*>(p.x + (size_t)row0 * p.inputs + kk) : zero;
      const uint4 x1 = in && row1 < p.tokens ? *reinterpret_cast<const uint4*>(p.x + (size_t)row1 * p.inputs + kk) : zero;
      const uint4 w = in ? *reinterpret_cast<const uint4*>(ar + kk) : zero;
      const uint32_t f0[4] = {x0.x, x1.x, x0.y, x1.y}, f1[4] = {x0.z, x1.z, x0.w, x1.w};
      mma_16816<true>(acc, f0, w.x, w.y);
      mma_16816<true>(acc, f1, w.z, w.w);
    }
    if (ids[g] == a) keep[0] = acc[0], keep[1] = acc[1];
    if (ids[g + 8] == a) keep[2] = acc[2], keep[3] = acc[3];
  }
  float* h = p.part + (size_t)blockIdx.y * p.tokens * R;
  const int c = r0 + 2 * t;
  if (row0 < p.tokens) *reinterpret_cast<float2*>(h + (size_t)row0 * R + c) = make_float2(keep[0], keep[1]);
  if (row1 < p.tokens) *reinterpret_cast<float2*>(h + (size_t)row1 * R + c) = make_float2(keep[2], keep[3]);
}

// (bf16(a), bf16(b)) and what is left of each, packed low = a
CCUT_DEVICE uint32_t take_bf16x2(float& a, float& b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  a -= __low2float(h);
  b -= __high2float(h);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Grid (tiles, blocks of 256 outputs): h of the tile in shared memory, summed over the splits and
// scaled; each warp takes 8 outputs at a time.  h enters the MMAs as bf16 parts whose sum keeps 16
// (two parts, bf16 output) or 24 (three, fp32 output) significant bits.
template <bool OUT_BF16>
__global__ void __launch_bounds__(kLoraWarps * 32) lora_expand_kernel(LoraArgs p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kParts = OUT_BF16 ? 2 : 3;
  __shared__ int ids[kLoraTile], uniq[kLoraTile], cnt;
  extern __shared__ float hs[];  // [16][R + 4]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int t0 = blockIdx.x * kLoraTile;
  const int n = tile_adapters(p, t0, ids, uniq, cnt);
  const int R = p.slices * p.rank, ld = R + 4;
  for (int i = threadIdx.x; i < kLoraTile * R; i += blockDim.x) {
    const int r = i / R, c = i % R, row = t0 + r, id = ids[r];
    float v = 0.f;
    if (id >= 0) {
      for (int s = 0; s < p.splits; ++s) v += p.part[((size_t)s * p.tokens + row) * R + c];
      v *= p.scales[id];
    }
    hs[r * ld + c] = v;
  }
  __syncthreads();
  const int row0 = t0 + g, row1 = t0 + g + 8;
  const int o_end = min(p.outputs, (int)(blockIdx.y + 1) * 256);
  for (int o = blockIdx.y * 256 + warp * 8; o < o_end; o += kLoraWarps * 8) {
    int j = 0;
    while (o >= p.ends[j]) ++j;  // slices end at multiples of 8: the eight outputs share one
    float keep[4] = {0.f, 0.f, 0.f, 0.f};
    for (int u = 0; u < n; ++u) {
      const int a = uniq[u];
      const uint16_t* br = p.b + ((size_t)a * p.outputs + o + g) * p.rank;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int k = 0; k < p.rank; k += 16) {
        const uint2 w = *reinterpret_cast<const uint2*>(br + k + 4 * t);
        const float* h0 = hs + g * ld + j * p.rank + k + 4 * t;
        float4 v0 = *reinterpret_cast<const float4*>(h0), v1 = *reinterpret_cast<const float4*>(h0 + 8 * ld);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          uint32_t f[4];
          f[0] = take_bf16x2(v0.x, v0.y);
          f[1] = take_bf16x2(v1.x, v1.y);
          f[2] = take_bf16x2(v0.z, v0.w);
          f[3] = take_bf16x2(v1.z, v1.w);
          mma_16816<true>(acc, f, w.x, w.y);
        }
      }
      if (ids[g] == a) keep[0] = acc[0], keep[1] = acc[1];
      if (ids[g + 8] == a) keep[2] = acc[2], keep[3] = acc[3];
    }
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int row = hi ? row1 : row0;
      if (row >= p.tokens) continue;
      const size_t bi = (size_t)row * p.base_ld + o + 2 * t, oi = (size_t)row * p.out_ld + o + 2 * t;
      const bool has = ids[g + 8 * hi] >= 0;
      if constexpr (OUT_BF16) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.base) + bi);
        const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(u << 16) + keep[2 * hi],
                                                       __uint_as_float(u & 0xFFFF0000u) + keep[2 * hi + 1]);
        *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + oi) =
            has ? *reinterpret_cast<const uint32_t*>(&v) : u;
      } else {
        const float2 u = *reinterpret_cast<const float2*>(static_cast<const float*>(p.base) + bi);
        *reinterpret_cast<float2*>(static_cast<float*>(p.out) + oi) =
            has ? make_float2(u.x + keep[2 * hi], u.y + keep[2 * hi + 1]) : u;
      }
    }
  }
}

static int lora_splits(int tokens, int inputs, int ranks) {
  const long base = (long)((tokens + kLoraTile - 1) / kLoraTile) * ((ranks + 31) / 32);
  long sp = base > 0 ? (2L * 148 + base - 1) / base : 1;
  const long most = (inputs + 127) / 128;
  if (sp > most) sp = most;
  if (sp > 32) sp = 32;
  return sp < 1 ? 1 : (int)sp;
}

}  // namespace ccut

using namespace ccut;

extern "C" {

size_t ccut_lora_workspace_bytes(int tokens, int inputs, int rank, int slices) {
  if (tokens < 0 || inputs <= 0 || rank <= 0 || slices <= 0 || (long)rank * slices > kLoraMaxRanks) return 0;
  return 256 + (size_t)lora_splits(tokens, inputs, rank * slices) * tokens * rank * slices * sizeof(float);
}

int ccut_lora_add(const uint16_t* x, const uint16_t* a, const uint16_t* b, const float* scales, const int32_t* ids,
                  int tokens, int inputs, int rank, int adapters, int slices, const int* widths, const void* base,
                  long long base_ld, void* out, long long out_ld, int dtype, void* workspace, size_t ws_bytes,
                  ccut_stream_t stream) {
  PdlScope pdl_scope(tokens);
  if (tokens < 0 || inputs <= 0 || inputs % 8 || rank <= 0 || rank % 16 || adapters < 0 || slices < 1 || !widths)
    return CCUT_ERR_INVALID;
  if (slices > CCUT_LORA_MAX_SLICES || (long)rank * slices > kLoraMaxRanks) return CCUT_ERR_UNSUPPORTED;
  if (dtype != CCUT_OUT_BF16 && dtype != CCUT_OUT_F32) return CCUT_ERR_INVALID;
  LoraArgs p{};
  long long o = 0;
  for (int j = 0; j < slices; ++j) {
    if (widths[j] <= 0 || widths[j] % 8) return CCUT_ERR_INVALID;
    o += widths[j];
    if (o > 2147483647LL - 256) return CCUT_ERR_UNSUPPORTED;
    p.ends[j] = (int)o;
  }
  if (base_ld < o || out_ld < o || base_ld % 8 || out_ld % 8) return CCUT_ERR_INVALID;
  if (tokens == 0) return CCUT_OK;
  if (!x || !ids || !base || !out || (adapters > 0 && (!a || !b || !scales))) return CCUT_ERR_INVALID;
  for (const void* q : {(const void*)x, (const void*)a, (const void*)b, base, (const void*)out})
    if (reinterpret_cast<uintptr_t>(q) % 16) return CCUT_ERR_INVALID;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      ws_bytes < ccut_lora_workspace_bytes(tokens, inputs, rank, slices))
    return CCUT_ERR_WORKSPACE;
  const int R = rank * slices;
  p.x = x, p.a = a, p.b = b, p.scales = scales, p.ids = ids;
  p.tokens = tokens, p.inputs = inputs, p.outputs = (int)o, p.rank = rank, p.slices = slices, p.adapters = adapters;
  p.base = base, p.base_ld = base_ld, p.out = out, p.out_ld = out_ld;
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256);
  p.splits = lora_splits(tokens, inputs, R);
  p.k_per_split = ((inputs + p.splits - 1) / p.splits + 31) / 32 * 32;
  const unsigned tiles = (tokens + kLoraTile - 1) / kLoraTile;
  int rc = launch_k(lora_shrink_kernel, dim3(tiles, p.splits, (R + 31) / 32), dim3(kLoraWarps * 32), 0, stream, p);
  if (rc) return rc;
  auto kern = dtype == CCUT_OUT_BF16 ? lora_expand_kernel<true> : lora_expand_kernel<false>;
  const size_t smem = (size_t)kLoraTile * (R + 4) * sizeof(float);
  const long long oblocks = (o + 255) / 256;
  if (oblocks > 65535) return CCUT_ERR_UNSUPPORTED;
  return launch_k(kern, dim3(tiles, (unsigned)oblocks), dim3(kLoraWarps * 32), smem, stream, p);
}

}  // extern "C"
