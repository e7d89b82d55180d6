// lora.cu -- low-rank adapters of many requests beside a shared projection.
//
//   out[t, o] = base[t, o] + scale[a] * sum_r B[a, o, r] * (sum_i A[a, j(o) rank + r, i] x[t, i]),  a = ids[t],
// where j(o) is the slice (q, k or v of a fused projection, say) that output o belongs to; a row whose
// id is outside [0, adapters) keeps its base.
//
// Two launches: lora_shrink_kernel writes partial products h[split, t, slices * rank] of the rows with their
// adapters' A, split over the inputs; lora_expand_kernel sums h in split order, scales it, multiplies by B
// and adds the base.  Both give a warp 16 tokens, the M of m16n8k16 bf16 MMAs, in one of two ways:
// - Up to kLoraGroupTokens tokens (a decode step), a CTA takes up to 16 tokens of ONE adapter, wherever they
//   are in the batch: every CTA sorts the few ids itself (each token's rank among its own), so that an
//   adapter's weights are read once however the requests mix, and all adapters at the same time.  Its four
//   warps split the inputs, then the outputs.  Bound: latency (two launches, three dependent loads each).
// - More tokens (prompts): a warp takes 16 neighbours and loops over their distinct adapters (one, inside a
//   prompt); the four warps of a CTA share its weights through the L1.  A row takes the result of its own
//   adapter by selection, so nothing of another request's adapter (a NaN weight, say) reaches it.  Bound: HBM
//   (x, base and out).
// Operands come straight from global memory: the order of the k index of an MMA is free, so a lane's operand
// registers are 16 consecutive bytes of a row of x or A (8 of B).  The outputs of two n-tiles interleave so
// that a lane holds four neighbours.
#include "host.cuh"

namespace ccut {

constexpr int kLoraTile = 16;   // tokens per warp
constexpr int kLoraWarps = 4;
constexpr int kLoraMaxRanks = 256;  // slices * rank
constexpr int kLoraGroupTokens = 256;
constexpr int kLoraRankTiles = 8;   // n-tiles of 8 rank rows a warp keeps
constexpr int kLoraOutputs = 512;   // outputs per CTA of the expand kernel (prompts)
constexpr int kLoraGroupOutputs = 256;

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

struct LoraTile {  // 16 rows and the adapters among them
  int rows[kLoraTile];  // tokens, -1: none
  int ids[kLoraTile];   // their adapters, -1: none
  int uniq[kLoraTile], n;
};

CCUT_DEVICE int lora_id(const LoraArgs& p, int t) {
  const int id = p.ids[t];
  return id >= 0 && id < p.adapters ? id : -1;
}

// Whole CTA (128 threads): the tile of unit `u` of the line of (id, up to 16 of its tokens), in order of first
// tokens; tokens without an adapter are units of id -1.  False past the last unit.
CCUT_DEVICE bool lora_group(const LoraArgs& p, int u, LoraTile& tile, int* ids, int* counts) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kPer = kLoraGroupTokens / (kLoraWarps * 32);
  for (int i = tid; i < kLoraGroupTokens; i += kLoraWarps * 32) ids[i] = i < p.tokens ? lora_id(p, i) : -2;
  if (tid < kLoraTile) tile.rows[tid] = -1, tile.ids[tid] = -1;
  if (tid == 0) tile.n = 0;
  __syncthreads();
  int mine[kPer], rank[kPer];
  unsigned leaders[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int t = tid + k * kLoraWarps * 32;
    mine[k] = ids[t];
    rank[k] = 0;
  }
  const int4* ids4 = reinterpret_cast<const int4*>(ids);
  for (int q = 0; q < (p.tokens + 3) / 4; ++q) {  // every token's rank among the tokens of its id
    const int4 v = ids4[q];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int t = tid + k * kLoraWarps * 32;
      rank[k] += (v.x == mine[k] && 4 * q < t) + (v.y == mine[k] && 4 * q + 1 < t) + (v.z == mine[k] && 4 * q + 2 < t) +
                 (v.w == mine[k] && 4 * q + 3 < t);
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    leaders[k] = __ballot_sync(0xffffffffu, mine[k] != -2 && rank[k] % kLoraTile == 0);
    if (lane == 0) counts[k * kLoraWarps + warp] = __popc(leaders[k]);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    int first = 0;
    for (int w = 0; w < k * kLoraWarps + warp; ++w) first += counts[w];
    if ((leaders[k] >> lane & 1) && first + __popc(leaders[k] & ((1u << lane) - 1)) == u) {
      tile.uniq[0] = mine[k];
      tile.uniq[1] = rank[k];
      tile.n = 1;
    }
  }
  __syncthreads();
  if (tile.n == 0) return false;
  const int id = tile.uniq[0], from = tile.uniq[1];
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (mine[k] == id && rank[k] >= from && rank[k] < from + kLoraTile) {
      tile.rows[rank[k] - from] = tid + k * kLoraWarps * 32;
      tile.ids[rank[k] - from] = id;
    }
  __syncthreads();
  return true;
}

// Whole warp: the tile of 16 neighbours from token t0.
CCUT_DEVICE void lora_neighbours(const LoraArgs& p, int t0, LoraTile& tile) {
  const int lane = threadIdx.x & 31, t = t0 + lane;
  const int id = lane < kLoraTile && t < p.tokens ? lora_id(p, t) : -1;
  const unsigned same = __match_any_sync(0xffffffffu, id);
  const bool first = id >= 0 && (same & ((1u << lane) - 1)) == 0;
  const unsigned firsts = __ballot_sync(0xffffffffu, first);
  if (lane < kLoraTile) {
    tile.rows[lane] = t < p.tokens ? t : -1;
    tile.ids[lane] = id;
    if (first) tile.uniq[__popc(firsts & ((1u << lane) - 1))] = id;
  }
  if (lane == 0) tile.n = __popc(firsts);
  __syncwarp();
}

// Grid (units or tiles of 64 tokens, splits, blocks of 64 rank rows).
template <bool GROUP>
__global__ void __launch_bounds__(kLoraWarps * 32) lora_shrink_kernel(const __grid_constant__ LoraArgs p) {
  pdl_wait();
  pdl_trigger();
  __shared__ LoraTile tiles[GROUP ? 1 : kLoraWarps];
  __shared__ __align__(16) int ids[GROUP ? kLoraGroupTokens : 4];
  __shared__ int counts[GROUP ? kLoraGroupTokens / 32 : 1];
  __shared__ float red[GROUP ? kLoraWarps - 1 : 1][GROUP ? 32 : 1][kLoraRankTiles * 4 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int R = p.slices * p.rank, r0 = blockIdx.z * kLoraRankTiles * 8;
  const int nz = min(kLoraRankTiles, (R - r0) / 8);
  LoraTile& tile = tiles[GROUP ? 0 : warp];
  int k0 = blockIdx.y * p.k_per_split, k1 = min(p.inputs, k0 + p.k_per_split);
  if constexpr (GROUP) {
    if (!lora_group(p, blockIdx.x, tile, ids, counts)) return;
    if (tile.uniq[0] < 0) return;
    const int per = p.k_per_split / kLoraWarps;  // a multiple of 32
    k0 += warp * per;
    k1 = min(k1, k0 + per);
  } else {
    lora_neighbours(p, (blockIdx.x * kLoraWarps + warp) * kLoraTile, tile);
  }
  const int row0 = tile.rows[g], row1 = tile.rows[g + 8];
  const uint16_t* x0 = p.x + (size_t)max(row0, 0) * p.inputs;
  const uint16_t* x1 = p.x + (size_t)max(row1, 0) * p.inputs;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  float keep[kLoraRankTiles][4];
#pragma unroll
  for (int n = 0; n < kLoraRankTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) keep[n][i] = 0.f;
  for (int u = 0; u < (GROUP ? 1 : tile.n); ++u) {
    const int a = tile.uniq[u];
    const uint16_t* ar = p.a + ((size_t)a * R + r0 + g) * p.inputs;
    float acc[kLoraRankTiles][4];
#pragma unroll
    for (int n = 0; n < kLoraRankTiles; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    // 32 inputs a step: lane t holds inputs k + 8 t .. + 7 of its rows
#pragma unroll 2
    for (int k = k0; k < k1; k += 32) {
      const int kk = k + 8 * t;
      const bool in = kk < k1;
      const uint4 v0 = in && row0 >= 0 ? __ldg(reinterpret_cast<const uint4*>(x0 + kk)) : zero;
      const uint4 v1 = in && row1 >= 0 ? __ldg(reinterpret_cast<const uint4*>(x1 + kk)) : zero;
      uint4 w[kLoraRankTiles];
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; ++n)
        w[n] = in && n < nz ? __ldg(reinterpret_cast<const uint4*>(ar + (size_t)n * 8 * p.inputs + kk)) : zero;
      const uint32_t f0[4] = {v0.x, v1.x, v0.y, v1.y}, f1[4] = {v0.z, v1.z, v0.w, v1.w};
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; ++n)
        if (n < nz) {
          mma_16816<true>(acc[n], f0, w[n].x, w[n].y);
          mma_16816<true>(acc[n], f1, w[n].z, w[n].w);
        }
    }
    const bool own0 = GROUP || tile.ids[g] == a, own1 = GROUP || tile.ids[g + 8] == a;
#pragma unroll
    for (int n = 0; n < kLoraRankTiles; ++n) {
      keep[n][0] = own0 ? acc[n][0] : keep[n][0];
      keep[n][1] = own0 ? acc[n][1] : keep[n][1];
      keep[n][2] = own1 ? acc[n][2] : keep[n][2];
      keep[n][3] = own1 ? acc[n][3] : keep[n][3];
    }
  }
  if constexpr (GROUP) {  // the warps' sums, in warp order
    if (warp > 0) {
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp - 1][lane][n * 4 + i] = keep[n][i];
    }
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 0; w < kLoraWarps - 1; ++w)
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[n][i] += red[w][lane][n * 4 + i];
  }
  float* h = p.part + (size_t)blockIdx.y * p.tokens * R + r0 + 2 * t;
#pragma unroll
  for (int n = 0; n < kLoraRankTiles; ++n)
    if (n < nz) {
      if (row0 >= 0) *reinterpret_cast<float2*>(h + (size_t)row0 * R + n * 8) = make_float2(keep[n][0], keep[n][1]);
      if (row1 >= 0) *reinterpret_cast<float2*>(h + (size_t)row1 * R + n * 8) = make_float2(keep[n][2], keep[n][3]);
    }
}

// (bf16(a), bf16(b)) and what is left of each, packed low = a
CCUT_DEVICE uint32_t take_bf16x2(float& a, float& b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  a -= __low2float(h);
  b -= __high2float(h);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four outputs of a row: base plus d (has: the row has an adapter).
template <bool BF16>
CCUT_DEVICE void lora_write(const LoraArgs& p, int row, int o, const float (&d)[4], bool has) {
  const size_t bi = (size_t)row * p.base_ld + o, oi = (size_t)row * p.out_ld + o;
  if constexpr (BF16) {
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p.base) + bi);
    const __nv_bfloat162 lo = __floats2bfloat162_rn(__uint_as_float(u.x << 16) + d[0], __uint_as_float(u.x & 0xFFFF0000u) + d[1]);
    const __nv_bfloat162 hi = __floats2bfloat162_rn(__uint_as_float(u.y << 16) + d[2], __uint_as_float(u.y & 0xFFFF0000u) + d[3]);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + oi) =
        has ? make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi)) : u;
  } else {
    const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(p.base) + bi);
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + oi) =
        has ? make_float4(u.x + d[0], u.y + d[1], u.z + d[2], u.w + d[3]) : u;
  }
}

// Grid (units or tiles of 64 tokens, blocks of outputs).  h enters the MMAs as bf16 parts whose sum keeps 16
// (two parts, bf16 output) or 24 (three, fp32 output) significant bits.  KR: rank / 16 when h's operands
// stay in registers for all outputs of a slice, 0 for other ranks.
template <bool GROUP, int KR, bool OUT_BF16>
__global__ void __launch_bounds__(kLoraWarps * 32) lora_expand_kernel(const __grid_constant__ LoraArgs p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kParts = OUT_BF16 ? 2 : 3;
  __shared__ LoraTile tiles[GROUP ? 1 : kLoraWarps];
  __shared__ __align__(16) int ids[GROUP ? kLoraGroupTokens : 4];
  __shared__ int counts[GROUP ? kLoraGroupTokens / 32 : 1];
  extern __shared__ __align__(16) float hs_all[];  // [1 or 4][16][R + 4]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int R = p.slices * p.rank, ld = R + 4;
  LoraTile& tile = tiles[GROUP ? 0 : warp];
  float* hs = hs_all + (GROUP ? 0 : warp * kLoraTile * ld);
  if constexpr (GROUP) {
    if (!lora_group(p, blockIdx.x, tile, ids, counts)) return;
    tile.n = tile.uniq[0] >= 0 ? 1 : 0;  // the same from every thread
  } else {
    lora_neighbours(p, (blockIdx.x * kLoraWarps + warp) * kLoraTile, tile);
  }
  if (p.base == p.out && tile.n == 0 && GROUP) return;  // in place: rows without an adapter stay
  for (int i = GROUP ? threadIdx.x : lane; i < kLoraTile * R / 4; i += GROUP ? kLoraWarps * 32 : 32) {
    const int r = i / (R / 4), c = i % (R / 4) * 4, row = tile.rows[r], id = tile.ids[r];
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (id >= 0) {
#pragma unroll 8
      for (int s = 0; s < p.splits; ++s) {
        const float4 y = *reinterpret_cast<const float4*>(p.part + ((size_t)s * p.tokens + row) * R + c);
        v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
      }
      const float f = p.scales[id];
      v.x *= f, v.y *= f, v.z *= f, v.w *= f;
    }
    *reinterpret_cast<float4*>(hs + r * ld + c) = v;
  }
  if constexpr (GROUP) __syncthreads();
  else __syncwarp();
  const int row0 = tile.rows[g], row1 = tile.rows[g + 8];
  const bool has0 = tile.ids[g] >= 0, has1 = tile.ids[g + 8] >= 0;
  // this warp's outputs, slice by slice
  constexpr int kWide = GROUP ? kLoraGroupOutputs / kLoraWarps : kLoraOutputs;
  const int o0 = GROUP ? blockIdx.y * kLoraGroupOutputs + warp * kWide : blockIdx.y * kWide;
  const int o1 = min(p.outputs, o0 + kWide);
  for (int j = 0; j < p.slices; ++j) {
    const int from = max(o0, j ? p.ends[j - 1] : 0), to = min(o1, p.ends[j]);
    if (from >= to) continue;
    uint32_t hf[KR ? KR : 1][kParts][4];
    auto operands = [&](int k, uint32_t(&f)[kParts][4]) {  // of rank columns 16 k ..: lane t takes 16 k + 4 t .. + 3
      const float* h0 = hs + g * ld + j * p.rank + 16 * k + 4 * t;
      float4 v0 = *reinterpret_cast<const float4*>(h0), v1 = *reinterpret_cast<const float4*>(h0 + 8 * ld);
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        f[part][0] = take_bf16x2(v0.x, v0.y);
        f[part][1] = take_bf16x2(v1.x, v1.y);
        f[part][2] = take_bf16x2(v0.z, v0.w);
        f[part][3] = take_bf16x2(v1.z, v1.w);
      }
    };
#pragma unroll
    for (int k = 0; k < KR; ++k) operands(k, hf[k]);
#pragma unroll 2
    for (int o = from; o < to; o += 16) {
      // n-tile i, column n is output o + 4 (n / 2) + 2 i + n % 2: lane t gets outputs o + 4 t .. + 3
      float keep[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      const int oc = o + (g >> 1) * 4 + (g & 1);
      for (int u = 0; u < tile.n; ++u) {
        const int a = tile.uniq[u];
        const uint16_t* br = p.b + ((size_t)a * p.outputs + oc) * p.rank + 4 * t;
        float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        auto product = [&](int k, const uint32_t(&f)[kParts][4]) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint2 w = oc + 2 * i < to ? __ldg(reinterpret_cast<const uint2*>(br + (size_t)2 * i * p.rank + 16 * k)) : make_uint2(0, 0);
#pragma unroll
            for (int part = 0; part < kParts; ++part) mma_16816<true>(acc[i], f[part], w.x, w.y);
          }
        };
        if constexpr (KR > 0) {
#pragma unroll
          for (int k = 0; k < KR; ++k) product(k, hf[k]);
        } else {
          for (int k = 0; k < p.rank / 16; ++k) {
            operands(k, hf[0]);
            product(k, hf[0]);
          }
        }
        const bool own0 = GROUP || tile.ids[g] == a, own1 = GROUP || tile.ids[g + 8] == a;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          keep[i][0] = own0 ? acc[i][0] : keep[i][0];
          keep[i][1] = own0 ? acc[i][1] : keep[i][1];
          keep[i][2] = own1 ? acc[i][2] : keep[i][2];
          keep[i][3] = own1 ? acc[i][3] : keep[i][3];
        }
      }
      if (o + 4 * t < to) {
        const float d0[4] = {keep[0][0], keep[0][1], keep[1][0], keep[1][1]};
        const float d1[4] = {keep[0][2], keep[0][3], keep[1][2], keep[1][3]};
        if (row0 >= 0) lora_write<OUT_BF16>(p, row0, o + 4 * t, d0, has0);
        if (row1 >= 0) lora_write<OUT_BF16>(p, row1, o + 4 * t, d1, has1);
      }
    }
  }
}

// Units of a decode step at most: one per adapter in use, one more per 16 tokens, tokens without one.
static int lora_units(int tokens, int adapters) {
  const long n = (long)adapters + 1 + tokens / kLoraTile;
  return (int)(n < tokens ? n : tokens);
}
// Splits of the inputs: two CTAs an SM for a decode step, four for prompts (whose loads in flight are what
// reads x fast), at least 128 inputs each.
static int lora_splits(int tokens, int inputs, int ranks, int adapters) {
  const bool group = tokens <= kLoraGroupTokens;
  const long z = (ranks + 8 * kLoraRankTiles - 1) / (8 * kLoraRankTiles);
  const long base = (group ? lora_units(tokens, adapters) : (tokens + 63) / 64) * z;
  long sp = base > 0 ? ((group ? 2L : 4L) * 148 + base - 1) / base : 1;
  const long most = (inputs + 127) / 128;
  if (sp > most) sp = most;
  if (sp > 16) sp = 16;
  return sp < 1 ? 1 : (int)sp;
}

template <bool GROUP, bool OB>
static int run_lora(const LoraArgs& p, cudaStream_t st) {
  const int R = p.rank * p.slices;
  const unsigned units = GROUP ? lora_units(p.tokens, p.adapters) : (p.tokens + 63) / 64;
  const unsigned z = (R + 8 * kLoraRankTiles - 1) / (8 * kLoraRankTiles);
  const dim3 block(kLoraWarps * 32);
  int rc = launch_k(lora_shrink_kernel<GROUP>, dim3(units, p.splits, z), block, 0, st, p);
  if (rc) return rc;
  const int wide = GROUP ? kLoraGroupOutputs : kLoraOutputs;
  const size_t smem = (size_t)(GROUP ? 1 : kLoraWarps) * kLoraTile * (R + 4) * sizeof(float);
  auto kern = p.rank == 16   ? lora_expand_kernel<GROUP, 1, OB>
              : p.rank == 32 ? lora_expand_kernel<GROUP, 2, OB>
              : p.rank == 64 ? lora_expand_kernel<GROUP, 4, OB>
                             : lora_expand_kernel<GROUP, 0, OB>;
  static std::atomic<uint64_t> smem_set[4];  // per kernel: devices with the limit raised
  const size_t most = (size_t)(GROUP ? 1 : kLoraWarps) * kLoraTile * (kLoraMaxRanks + 4) * sizeof(float);
  rc = ensure_smem_limit(kern, most, smem_set[p.rank == 16 ? 0 : p.rank == 32 ? 1 : p.rank == 64 ? 2 : 3]);
  if (rc) return rc;
  return launch_k(kern, dim3(units, (unsigned)((p.outputs + wide - 1) / wide)), block, smem, st, p);
}

}  // namespace ccut

using namespace ccut;

extern "C" {

size_t ccut_lora_workspace_bytes(int tokens, int inputs, int rank, int slices, int adapters) {
  if (tokens < 0 || inputs <= 0 || rank <= 0 || slices <= 0 || adapters < 0 || (long)rank * slices > kLoraMaxRanks)
    return 0;
  return 256 + (size_t)lora_splits(tokens, inputs, rank * slices, adapters) * tokens * rank * slices * sizeof(float);
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
  if (base_ld < o || out_ld < o || base_ld % 8 || out_ld % 8 || (base == out && base_ld != out_ld))
    return CCUT_ERR_INVALID;
  if (tokens == 0) return CCUT_OK;
  if (!x || !ids || !base || !out || (adapters > 0 && (!a || !b || !scales))) return CCUT_ERR_INVALID;
  for (const void* q : {(const void*)x, (const void*)a, (const void*)b, base, (const void*)out})
    if (reinterpret_cast<uintptr_t>(q) % 16) return CCUT_ERR_INVALID;
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      ws_bytes < ccut_lora_workspace_bytes(tokens, inputs, rank, slices, adapters))
    return CCUT_ERR_WORKSPACE;
  const int R = rank * slices;
  p.x = x, p.a = a, p.b = b, p.scales = scales, p.ids = ids;
  p.tokens = tokens, p.inputs = inputs, p.outputs = (int)o, p.rank = rank, p.slices = slices, p.adapters = adapters;
  p.base = base, p.base_ld = base_ld, p.out = out, p.out_ld = out_ld;
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256);
  p.splits = lora_splits(tokens, inputs, R, adapters);
  const int step = tokens <= kLoraGroupTokens ? 32 * kLoraWarps : 32;  // each warp takes whole steps of 32
  p.k_per_split = ((inputs + p.splits - 1) / p.splits + step - 1) / step * step;
  if ((o + kLoraGroupOutputs - 1) / kLoraGroupOutputs > 65535) return CCUT_ERR_UNSUPPORTED;
  const bool ob = dtype == CCUT_OUT_BF16;
  if (tokens <= kLoraGroupTokens) return ob ? run_lora<true, true>(p, stream) : run_lora<true, false>(p, stream);
  return ob ? run_lora<false, true>(p, stream) : run_lora<false, false>(p, stream);
}

}  // extern "C"
