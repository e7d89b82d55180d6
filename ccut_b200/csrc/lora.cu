// lora.cu -- low-rank adapters of many requests beside a shared projection.
//
//   out[t, o] = base[t, o] + scale[a] * sum_r B[a, o, r] * (sum_i A[a, j(o) rank + r, i] x[t, i]),  a = ids[t],
// where j(o) is the slice (q, k or v of a fused projection, say) that output o belongs to; a row whose
// id is outside [0, adapters) keeps its base.
//
// Products are m16n8k16 bf16 MMAs with 16 tokens as the M, in one of two ways:
// - Up to kLoraGroupTokens tokens (a decode step), one launch: a cluster takes up to 16 tokens of ONE adapter,
//   wherever they are in the batch: every CTA sorts the few ids itself (each token's rank among its own), so that
//   an adapter's weights are read once however the requests mix, and all adapters at the same time.  Bound:
//   latency.  The CTAs and warps split the inputs, add up h through distributed shared memory and then split
//   the outputs; operands come straight from global memory (the order of the k index of an MMA is free: a
//   lane's operand registers are 16 consecutive bytes of a row of x or A).
//   64 tokens, 16 adapters of rank 16, 2048 inputs, 5120 outputs: 10.3 us (14.8 in two kernels that
//   passed h through memory; one token alone: 7.7 and 5.8, but a launch less is 4 us less of host time).
// - More tokens (prompts), two launches: a shrink kernel gives h[t, slices * rank] = A x, the expand kernel scales it,
//   multiplies by B and adds the base.  A CTA takes 64 neighbours and loops over their distinct adapters (one,
//   inside a prompt).  A row takes the result of its own adapter by selection, so nothing of another request's
//   adapter (a NaN weight, say) reaches it.  x and A stream through a cp.async ring; the inputs are split
//   over a cluster of up to 8 CTAs whose sums meet in distributed shared memory, in rank order.  Bound: HBM (x, base
//   and out).  4093 tokens, rank 64, 4096 inputs, 2048 bf16 outputs: 38 us, 1.8 TB/s
//   (18 + 20: a CTA's few stages are mostly their latency).
// The outputs of two n-tiles interleave so that a lane holds four neighbours.
#include <type_traits>

#include "host.cuh"
#include "tc.cuh"

namespace ccut {

constexpr int kLoraTile = 16;   // tokens per warp
constexpr int kLoraWarps = 4;
constexpr int kLoraMaxRanks = 256;  // slices * rank
constexpr int kLoraGroupTokens = 256;
constexpr int kLoraRankTiles = 8;   // n-tiles of 8 rank rows a warp keeps
constexpr int kLoraRows = kLoraTile * kLoraWarps;  // tokens per CTA (prompts)
constexpr int kLoraStep = 64;       // inputs per stage of the ring
constexpr int kLoraStages = 3;
constexpr int kLoraOutputs = 128;   // outputs per CTA of the expand kernels

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
#pragma unroll 4
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
#pragma unroll
    for (int w = 0; w < kLoraGroupTokens / 32; ++w) first += w < k * kLoraWarps + warp ? counts[w] : 0;
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

// 64 neighbours and the adapters among them.
struct LoraRows {
  int ids[kLoraRows];   // -1: none, or past the last token
  int uniq[kLoraRows], n;
};
// Whole CTA.
CCUT_DEVICE void lora_neighbours(const LoraArgs& p, int t0, LoraRows& rows) {
  const int tid = threadIdx.x;
  if (tid < kLoraRows) rows.ids[tid] = t0 + tid < p.tokens ? lora_id(p, t0 + tid) : -1;
  __syncthreads();
  if (tid < 32) {  // first of their kind, in order
    int n = 0;
#pragma unroll
    for (int k = 0; k < kLoraRows; k += 32) {
      const int id = rows.ids[k + tid];
      const unsigned same = __match_any_sync(0xffffffffu, id);  // every lane takes part
      bool first = id >= 0 && (same & ((1u << tid) - 1)) == 0;
      if (k > 0)
        for (int i = 0; i < n; ++i) first &= rows.uniq[i] != id;
      const unsigned m = __ballot_sync(0xffffffffu, first);
      if (first) rows.uniq[n + __popc(m & ((1u << tid) - 1))] = id;
      n += __popc(m);
      __syncwarp();
    }
    if (tid == 0) rows.n = n;
  }
  __syncthreads();
}

// Byte offset of 16-byte chunk c of row r in a tile of 128-byte rows: ldmatrix reads 8 rows of one chunk without
// meeting a bank twice.
CCUT_DEVICE int lora_chunk(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
CCUT_DEVICE void lora_copy(uint32_t to, const void* from, bool in) {  // 16 bytes, zeros when !in
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}
CCUT_DEVICE void st_cluster(uint32_t addr, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
CCUT_DEVICE float4 ld_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Prompts.  Grid (tiles of 64 tokens, splits, blocks of 64 rank rows), the splits of a tile in one cluster.
constexpr int kLoraStageBytes = 2 * kLoraRows * kLoraStep * 2;  // x and A, 64 rows of 128 bytes each
__global__ void __launch_bounds__(kLoraWarps * 32) lora_shrink_kernel(const __grid_constant__ LoraArgs p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ LoraRows rows;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int R = p.slices * p.rank, r0 = blockIdx.z * kLoraRankTiles * 8;
  const int nz = min(kLoraRankTiles, (R - r0) / 8), t0 = blockIdx.x * kLoraRows;
  const int k0 = blockIdx.y * p.k_per_split, k1 = min(p.inputs, k0 + p.k_per_split);
  const int steps = k1 > k0 ? (k1 - k0 + kLoraStep - 1) / kLoraStep : 0;
  // copies of a stage: thread -> 16-byte chunk tid % 8 of rows tid / 8, + 16, + 32, + 48 of x and of A; the
  // addresses move from stage to stage and back at the next adapter
  const int cr = threadIdx.x >> 3, cc = threadIdx.x & 7;
  const int first_k = k0 + cc * 8;
  const uint16_t* xa = p.x + (size_t)min(t0 + cr, p.tokens - 1) * p.inputs;
  const size_t hop = (size_t)16 * p.inputs;
  int fetch_step = 0, fetch_adapter = 0, fetch_stage = 0, fetch_k = first_k;
  const uint16_t* wa = nullptr;
  const int xrows = (p.tokens - t0 - cr + 15) / 16, wrows = (nz * 8 - cr + 15) / 16;  // of the four, those that exist
  const uint32_t to = smem_u32(ring) + lora_chunk(cr, cc);  // rows 16 apart: the same place, 2048 bytes on
  auto issue_x = [&](int stage, int k) {
#pragma unroll
    for (int i = 0; i < kLoraRows / 16; ++i) {
      const bool in = k < k1 && i < xrows;
      lora_copy(to + stage * kLoraStageBytes + i * 2048, in ? xa + i * hop + k : p.x, in);
    }
  };
  auto issue = [&](bool with_x) {
    if (fetch_step == 0) wa = p.a + ((size_t)rows.uniq[fetch_adapter] * R + r0 + min(cr, nz * 8 - 1)) * p.inputs;
    if (with_x) issue_x(fetch_stage, fetch_k);
#pragma unroll
    for (int i = 0; i < kLoraRows / 16; ++i) {
      const bool in = fetch_k < k1 && i < wrows;
      lora_copy(to + fetch_stage * kLoraStageBytes + kLoraRows * 128 + i * 2048, in ? wa + i * hop + fetch_k : p.x, in);
    }
    fetch_k += kLoraStep;
    if (++fetch_stage == kLoraStages) fetch_stage = 0;
    if (++fetch_step == steps) fetch_step = 0, ++fetch_adapter, fetch_k = first_k;
  };
#pragma unroll
  for (int i = 0; i < kLoraStages - 1; ++i)
    if (i < steps) issue_x(i, first_k + i * kLoraStep);  // on its way during the lookup
  lora_neighbours(p, t0, rows);
  const int total = steps * rows.n;
  float keep[kLoraRankTiles][4], acc[kLoraRankTiles][4];
#pragma unroll
  for (int n = 0; n < kLoraRankTiles; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) keep[n][i] = 0.f, acc[n][i] = 0.f;
  const int id0 = rows.ids[warp * kLoraTile + g], id1 = rows.ids[warp * kLoraTile + g + 8];
#pragma unroll
  for (int i = 0; i < kLoraStages - 1; ++i) {
    if (i < total) issue(i >= steps);
    cp_async_commit();
  }
  int step = 0, adapter = 0, stage = 0;
  for (int s = 0; s < total; ++s) {
    cp_async_wait<kLoraStages - 2>();
    __syncthreads();  // everyone's copies of this stage have landed, everyone is done with the stage before
    if (s + kLoraStages - 1 < total) issue(true);
    cp_async_commit();
    const uint8_t* st = ring + stage * kLoraStageBytes;
    if (++stage == kLoraStages) stage = 0;
#pragma unroll
    for (int kk = 0; kk < kLoraStep / 16; ++kk) {
      uint32_t f[4];
      ldmatrix_x4(f[0], f[1], f[2], f[3], st + lora_chunk(warp * kLoraTile + (lane & 15), kk * 2 + (lane >> 4)));
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; n += 2)
        if (n < nz) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4(b0, b1, b2, b3,
                      st + kLoraRows * 128 + lora_chunk(n * 8 + (lane & 7) + (lane >> 4) * 8, kk * 2 + (lane >> 3 & 1)));
          mma_16816<true>(acc[n], f, b0, b1);
          mma_16816<true>(acc[n + 1], f, b2, b3);
        }
    }
    if (++step == steps) {  // the last of an adapter: its rows take the sums
      const int a = rows.uniq[adapter++];
      step = 0;
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; ++n) {
        keep[n][0] = id0 == a ? acc[n][0] : keep[n][0];
        keep[n][1] = id0 == a ? acc[n][1] : keep[n][1];
        keep[n][2] = id1 == a ? acc[n][2] : keep[n][2];
        keep[n][3] = id1 == a ? acc[n][3] : keep[n][3];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();
  // sums of this CTA in its shared memory, [64 tokens][64 rank rows + 4], then each CTA of the cluster adds up its
  // share of the tokens over all, in rank order
  constexpr int kLd = kLoraRankTiles * 8 + 4;
  float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int n = 0; n < kLoraRankTiles; ++n) {
    float* d = sums + (warp * kLoraTile + g) * kLd + n * 8 + 2 * t;
    d[0] = keep[n][0], d[1] = keep[n][1];
    d[8 * kLd] = keep[n][2], d[8 * kLd + 1] = keep[n][3];
  }
  __syncthreads();
  tc::cluster_sync();
  const int share = kLoraRows / p.splits;
  for (int i = threadIdx.x; i < share * (nz * 2); i += kLoraWarps * 32) {
    const int r = blockIdx.y * share + i / (nz * 2), c = i % (nz * 2) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < p.splits; ++s) {
      const float4 y = ld_cluster(tc::mapa(sums + r * kLd + c, s));
      v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
    }
    if (t0 + r < p.tokens) *reinterpret_cast<float4*>(p.part + (size_t)(t0 + r) * R + r0 + c) = v;
  }
  __syncthreads();
  tc::cluster_sync();  // no CTA leaves while its sums are read
}

// (bf16(a), bf16(b)) and what is left of each, packed low = a
CCUT_DEVICE uint32_t take_bf16x2(float& a, float& b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  a -= __low2float(h);
  b -= __high2float(h);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Four neighbouring values of a row of base (or out).
template <bool BF16>
struct LoraFour {
  using Raw = typename std::conditional<BF16, uint2, float4>::type;
  static CCUT_DEVICE Raw load(const void* p, size_t at) {
    if constexpr (BF16) return *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + at);
    else return *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
  }
  static CCUT_DEVICE void store(void* p, size_t at, const Raw& v) {
    if constexpr (BF16) *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + at) = v;
    else *reinterpret_cast<float4*>(static_cast<float*>(p) + at) = v;
  }
  static CCUT_DEVICE Raw add(const Raw& u, float a, float b, float c, float d) {  // the one rounding
    if constexpr (BF16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(__uint_as_float(u.x << 16) + a, __uint_as_float(u.x & 0xFFFF0000u) + b);
      const __nv_bfloat162 hi = __floats2bfloat162_rn(__uint_as_float(u.y << 16) + c, __uint_as_float(u.y & 0xFFFF0000u) + d);
      return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      return make_float4(u.x + a, u.y + b, u.z + c, u.w + d);
    }
  }
};

// h enters the MMAs as bf16 parts whose sum keeps 16 (two parts, bf16 output) or 24 (three, fp32 output)
// significant bits, kept as planes [part][rows][lora_ld(R)] in shared memory.
// Rows of the planes and of B are an odd multiple of 32 bytes apart: the 8 bytes of 4 lanes x 4 rows that half a
// warp reads meet every bank once.
__host__ __device__ constexpr int lora_ld(int n) { return n % 32 ? n : n + 16; }  // n a multiple of 16 elements
template <int kParts>
CCUT_DEVICE void lora_keep(uint16_t* planes, size_t plane, size_t at, float4 v) {
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    const uint32_t lo = take_bf16x2(v.x, v.y), hi = take_bf16x2(v.z, v.w);
    *reinterpret_cast<uint2*>(planes + part * plane + at) = make_uint2(lo, hi);
  }
}
// Operand parts of rank columns `at` .. + 3 of rows g (h0) and g + 8.
template <int kParts>
CCUT_DEVICE void lora_operands(const uint16_t* h0, size_t plane, int ld, uint32_t (&f)[kParts][4]) {
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    const uint2 u = *reinterpret_cast<const uint2*>(h0 + part * plane);
    const uint2 v = *reinterpret_cast<const uint2*>(h0 + part * plane + 8 * ld);
    f[part][0] = u.x, f[part][1] = v.x, f[part][2] = u.y, f[part][3] = v.y;
  }
}

// Slice of output o.
CCUT_DEVICE int lora_slice(const LoraArgs& p, int o) {
  int j = 0;
#pragma unroll
  for (int i = 0; i < CCUT_LORA_MAX_SLICES - 1; ++i) j += i + 1 < p.slices && o >= p.ends[i];
  return j;
}

// Decode steps.  Grid (C, units), a cluster of C = p.splits CTAs per unit.  The CTAs split the inputs; their sums of h
// meet in every CTA through distributed shared memory, in rank order, and the warps of the cluster then take the
// outputs in turn, in blocks of 8 x 2 (column n of n-tile i: output 4 (n / 2) + 2 i + n % 2 of 16; slices end at
// multiples of 8, so a block of 16 has one or two).
__host__ __device__ constexpr int lora_hp_ld(int R) { return R + 4; }
__host__ __device__ constexpr size_t lora_group_smem(int R, int parts) {
  const size_t planes = (size_t)parts * kLoraTile * lora_ld(R) * 2, red = (size_t)(kLoraWarps - 1) * 32 * (kLoraRankTiles * 4 + 1) * 4;
  return (size_t)kLoraTile * lora_hp_ld(R) * 4 + (planes > red ? planes : red);
}
template <bool OUT_BF16, int kBlocks, int kFetch>
__global__ void __launch_bounds__(kLoraWarps * 32, 3) lora_group_kernel(const __grid_constant__ LoraArgs p) {
  pdl_wait();
  pdl_trigger();
  constexpr int kParts = OUT_BF16 ? 2 : 3;
  using Four = LoraFour<OUT_BF16>;
  __shared__ LoraTile tile;
  __shared__ __align__(16) int ids[kLoraGroupTokens];
  __shared__ int counts[kLoraGroupTokens / 32];
  extern __shared__ __align__(16) float hp[];  // [16][R + 4] this CTA's sums; then the warps' sums, later the planes of h
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int R = p.slices * p.rank, ld = lora_ld(R), hld = lora_hp_ld(R), part = blockIdx.x;
  const size_t plane = (size_t)kLoraTile * ld;
  float(*red)[32][kLoraRankTiles * 4 + 1] = reinterpret_cast<float(*)[32][kLoraRankTiles * 4 + 1]>(hp + kLoraTile * hld);
  uint16_t* hs = reinterpret_cast<uint16_t*>(hp + kLoraTile * hld);  // [parts][16][lora_ld(R)]
  if (!lora_group(p, blockIdx.y, tile, ids, counts)) return;  // the same for the whole cluster, as the next
  const int a = tile.uniq[0];
  if (a < 0 && p.base == p.out) return;  // in place: rows without an adapter stay
  const int row0 = tile.rows[g], row1 = tile.rows[g + 8];

  if (a >= 0) {  // h of this CTA's inputs
    // up to 64 rank rows a warp: the warps split the rank rows first, the inputs where there are fewer
    static_assert(kLoraWarps == 4, "");
    const int shift = R <= 8 * kLoraRankTiles ? 0 : R <= 16 * kLoraRankTiles ? 1 : 2, rw = 1 << shift;
    const int wr = warp & (rw - 1), wk = warp >> shift, r0 = wr * kLoraRankTiles * 8, nz = min(kLoraRankTiles, (R - r0) / 8);
    const int per = p.k_per_split >> (2 - shift);  // a multiple of 32
    const int k0 = part * p.k_per_split + wk * per, k1 = nz > 0 ? min(p.inputs, k0 + per) : k0;
    const uint16_t* x0 = p.x + (size_t)max(row0, 0) * p.inputs;
    const uint16_t* x1 = p.x + (size_t)max(row1, 0) * p.inputs;
    const uint16_t* ar = p.a + ((size_t)a * R + r0 + g) * p.inputs;
    const uint4 zero = make_uint4(0, 0, 0, 0);
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
    if (wk > 0) {  // the warps' sums, in the order of their inputs
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp - rw][lane][n * 4 + i] = acc[n][i];
    }
    __syncthreads();
    if (wk == 0) {
      for (int w = wr; w < kLoraWarps - rw; w += rw)
#pragma unroll
        for (int n = 0; n < kLoraRankTiles; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[n][i] += red[w][lane][n * 4 + i];
#pragma unroll
      for (int n = 0; n < kLoraRankTiles; ++n)
        if (n < nz) {
          float* h = hp + r0 + n * 8 + 2 * t;
          *reinterpret_cast<float2*>(h + g * hld) = make_float2(acc[n][0], acc[n][1]);
          *reinterpret_cast<float2*>(h + (g + 8) * hld) = make_float2(acc[n][2], acc[n][3]);
        }
    }
  }

  // this warp's blocks of 16 outputs, kBlocks at a time: base and kFetch k steps of B on their way before they are
  // needed
  const int blocks = (p.outputs + 15) / 16, stride = p.splits * kLoraWarps, steps = p.rank / 16;
  typename Four::Raw base[kBlocks][2];
  uint2 w[kBlocks][2][kFetch];
  auto fetch = [&](int block) {
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
      const int o16 = (block + q * stride) * 16, o = o16 + 4 * t, oc = o16 + (g >> 1) * 4 + (g & 1);
      if (o < p.outputs) {
        if (row0 >= 0) base[q][0] = Four::load(p.base, (size_t)row0 * p.base_ld + o);
        if (row1 >= 0) base[q][1] = Four::load(p.base, (size_t)row1 * p.base_ld + o);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < kFetch; ++k)
          w[q][i][k] = a >= 0 && oc + 2 * i < p.outputs && k < steps
                           ? __ldg(reinterpret_cast<const uint2*>(p.b + ((size_t)a * p.outputs + oc + 2 * i) * p.rank + 16 * k + 4 * t))
                           : make_uint2(0, 0);
    }
  };
  const int block0 = part * kLoraWarps + warp;
  fetch(block0);
  if (a >= 0) {
    // each CTA adds up its share of h and puts the sums in their place in all (every CTA adding up all of h took 9000
    // cycles with 16 of them)
    const int all = kLoraTile * R / 4, share = (all + p.splits - 1) / p.splits, end = min(all, (part + 1) * share);
    tc::cluster_sync();
    for (int i = part * share + threadIdx.x; i < end; i += kLoraWarps * 32) {
      const float* at = hp + i / (R / 4) * hld + i % (R / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int s = 0; s < p.splits; ++s) {
        const float4 y = ld_cluster(tc::mapa(at, s));
        v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
      }
      for (int s = 0; s < p.splits; ++s) st_cluster(tc::mapa(at, s), v);
    }
    tc::cluster_sync();
    const float scale = p.scales[a];
    for (int i = threadIdx.x; i < all; i += kLoraWarps * 32) {
      const int r = i / (R / 4), c = i % (R / 4) * 4;
      const float4 v = *reinterpret_cast<const float4*>(hp + r * hld + c);
      lora_keep<kParts>(hs, plane, r * ld + c, make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale));
    }
    __syncthreads();
  }
  for (int block = block0; block < blocks; block += kBlocks * stride) {
    if (block > block0) fetch(block);
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) {
      const int o = (block + q * stride) * 16;
      if (o >= p.outputs) break;
      float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if (a >= 0) {
        // both halves of the block (8 outputs, lanes t < 2 and t >= 2) share a slice, or each has its own
        const int j0 = lora_slice(p, o), j1 = o + 8 < p.outputs ? lora_slice(p, o + 8) : j0;
        const int oc = o + (g >> 1) * 4 + (g & 1);
        for (int j = j0; j <= j1; ++j) {
          float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
          const uint16_t* h = hs + g * ld + j * p.rank + 4 * t;
          auto step = [&](int k, uint2 b0, uint2 b1) {
            uint32_t f[kParts][4];
            lora_operands<kParts>(h + 16 * k, plane, ld, f);
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              mma_16816<true>(acc[0], f[part], b0.x, b0.y);
              mma_16816<true>(acc[1], f[part], b1.x, b1.y);
            }
          };
#pragma unroll
          for (int k = 0; k < kFetch; ++k)
            if (k < steps) step(k, w[q][0][k], w[q][1][k]);
          for (int k = kFetch; k < steps; ++k) {
            uint2 b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              b[i] = oc + 2 * i < p.outputs
                         ? __ldg(reinterpret_cast<const uint2*>(p.b + ((size_t)a * p.outputs + oc + 2 * i) * p.rank + 16 * k + 4 * t))
                         : make_uint2(0, 0);
            step(k, b[0], b[1]);
          }
          const bool mine = (t < 2 ? j0 : j1) == j;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i][e] = mine ? acc[i][e] : d[i][e];
        }
      }
      if (o + 4 * t < p.outputs) {
        const bool has = a >= 0;
        if (row0 >= 0)
          Four::store(p.out, (size_t)row0 * p.out_ld + o + 4 * t,
                      has ? Four::add(base[q][0], d[0][0], d[0][1], d[1][0], d[1][1]) : base[q][0]);
        if (row1 >= 0)
          Four::store(p.out, (size_t)row1 * p.out_ld + o + 4 * t,
                      has ? Four::add(base[q][1], d[0][2], d[0][3], d[1][2], d[1][3]) : base[q][1]);
      }
    }
  }
}

// Where output r of a block lies in shared memory: column n of n-tile i at 16-block + 8 i + n.
CCUT_DEVICE int lora_place(int r) { return (r & ~15) + ((r >> 1) & 1) * 8 + ((r >> 2) & 3) * 2 + (r & 1); }

// Prompts.  Grid (tiles of 64 tokens, blocks of 128 outputs): base is on its way while the adapters are looked up,
// the adapter's rows of B next, all before the wait for h; warp w has tokens 16 w .. and all the outputs.  KR: rank / 16, or
// 0 for any.
template <int KR, bool OUT_BF16>
__global__ void __launch_bounds__(kLoraWarps * 32, OUT_BF16 ? 4 : 3)
    lora_expand_kernel(const __grid_constant__ LoraArgs p) {
  constexpr int kParts = OUT_BF16 ? 2 : 3, kBlocks = kLoraOutputs / 16;
  using Four = LoraFour<OUT_BF16>;
  __shared__ LoraRows rows;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int R = p.slices * p.rank, ld = lora_ld(R), steps = KR ? KR : p.rank / 16;
  const int bld = lora_ld(p.rank) * 2;  // bytes per row of B
  const size_t plane = (size_t)kLoraRows * ld;
  constexpr bool kRegs = KR > 0;  // h of a slice fits registers, as operands; else planes in shared memory
  uint16_t* hs = reinterpret_cast<uint16_t*>(smem);             // [parts][64][lora_ld(R)]
  uint8_t* bs = smem + (kRegs ? 0 : kParts * plane * 2);        // [128][rank] bf16
  // base, then out: [64][128], moved 16 bytes a lane, whole lines at a time
  constexpr int kSize = OUT_BF16 ? 2 : 4, kOld = kLoraOutputs * kSize + 16 * kSize, kChunks = kLoraOutputs * kSize / 16;
  uint8_t* os = bs + kLoraOutputs * bld;
  const int t0 = blockIdx.x * kLoraRows, o0 = blockIdx.y * kLoraOutputs, width = min(kLoraOutputs, p.outputs - o0);
  const int row0 = t0 + warp * kLoraTile + g, row1 = row0 + 8;
  const bool in0 = row0 < p.tokens, in1 = row1 < p.tokens;
  // h of rows g and g + 8, columns 4 t + 16 c .. + 3 (rows without an adapter are zeros there)
  constexpr int kBatch = kRegs ? KR : 4;
  float4 h[2][kBatch];
  auto load_h = [&](int c0) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < kBatch; ++c)
        h[i][c] = (i ? in1 : in0) && (c0 + c) * 16 < R
                      ? *reinterpret_cast<const float4*>(p.part + (size_t)(i ? row1 : row0) * R + (c0 + c) * 16 + 4 * t)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  int slice = kRegs ? lora_slice(p, o0) : 0;  // whose h is in registers
  constexpr int kHop = kLoraWarps * 32 / kChunks;  // rows that the CTA moves at a time
  const int mr = threadIdx.x / kChunks, mc = threadIdx.x % kChunks;
  const bool mine = mc < width * kSize / 16;  // widths are multiples of 8: whole chunks
  const int mrows = mine ? min(kLoraRows, p.tokens - t0) : 0;
  {
    const uint8_t* from = static_cast<const uint8_t*>(p.base) + ((size_t)(t0 + mr) * p.base_ld + o0) * kSize + mc * 16;
    const size_t hop = (size_t)kHop * p.base_ld * kSize;
    const uint32_t to = smem_u32(os) + mr * kOld + mc * 16;
#pragma unroll
    for (int r = 0; r < kLoraRows; r += kHop)
      if (r + mr < mrows) lora_copy(to + r * kOld, from + r / kHop * hop, true);
  }
  cp_async_commit();
  lora_neighbours(p, t0, rows);
  auto fetch_b = [&](int a) {
    const int br = threadIdx.x >> 3, bc = threadIdx.x & 7;
    const uint16_t* from = p.b + ((size_t)a * p.outputs + o0 + br) * p.rank + bc * 8;
    const uint32_t to = smem_u32(bs) + lora_place(br) * bld + bc * 16;
#pragma unroll
    for (int r = 0; r < kLoraOutputs; r += 16)
      if (r + br < width)
        for (int c = 0; c < p.rank / 8 - bc; c += 8) lora_copy(to + r * bld + c * 16, from + (size_t)r * p.rank + c * 8, true);
    cp_async_commit();
  };
  if (rows.n > 0) fetch_b(rows.uniq[0]);
  pdl_wait();  // base, ids and B were there before the shrink kernel began; h is what it makes
  pdl_trigger();
  load_h(slice * KR);
  const int id0 = rows.ids[warp * kLoraTile + g], id1 = rows.ids[warp * kLoraTile + g + 8];
  const float f0 = id0 >= 0 ? p.scales[id0] : 0.f, f1 = id1 >= 0 ? p.scales[id1] : 0.f;
  uint32_t hf[kRegs ? KR : 1][kParts][4];
  auto keep_h = [&]() {  // scaled, in parts
#pragma unroll
    for (int c = 0; c < kBatch; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float f = i ? f1 : f0;
        float4 v = make_float4(h[i][c].x * f, h[i][c].y * f, h[i][c].z * f, h[i][c].w * f);
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          hf[c][part][i] = take_bf16x2(v.x, v.y);
          hf[c][part][i + 2] = take_bf16x2(v.z, v.w);
        }
      }
  };
  if constexpr (kRegs) keep_h();
  for (int c0 = 0; !kRegs && c0 * 16 < R; c0 += kBatch) {
    if (c0 > 0) load_h(c0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < kBatch; ++c)
        if ((c0 + c) * 16 < R) {
          const float f = i ? f1 : f0;
          const float4 v = make_float4(h[i][c].x * f, h[i][c].y * f, h[i][c].z * f, h[i][c].w * f);
          lora_keep<kParts>(hs, plane, (warp * kLoraTile + g + 8 * i) * ld + (c0 + c) * 16 + 4 * t, v);
        }
  }
  for (int u = 0; u < rows.n; ++u) {
    const int a = rows.uniq[u];
    cp_async_wait<0>();
    __syncthreads();
    if (__any_sync(0xffffffffu, id0 == a || id1 == a)) {
#pragma unroll
      for (int q = 0; q < kBlocks; ++q) {
        const int o = o0 + q * 16;
        if (o >= p.outputs) break;
        float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        const int j0 = lora_slice(p, o), j1 = o + 8 < p.outputs ? lora_slice(p, o + 8) : j0;
        const uint8_t* br = bs + (q * 16 + g) * bld + 8 * t;
        for (int j = j0; j <= j1; ++j) {
          float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
          const uint16_t* hr = hs + (warp * kLoraTile + g) * ld + j * p.rank + 4 * t;
          if constexpr (kRegs) {
            if (j != slice) {
              slice = j;
              load_h(j * KR);
              keep_h();
            }
          }
#pragma unroll KR ? KR : 1
          for (int k = 0; k < steps; ++k) {
            uint32_t f[kParts][4];
            if constexpr (kRegs) {
#pragma unroll
              for (int part = 0; part < kParts; ++part)
#pragma unroll
                for (int e = 0; e < 4; ++e) f[part][e] = hf[k][part][e];
            } else {
              lora_operands<kParts>(hr + 16 * k, plane, ld, f);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // a column past the last output is not written, whatever it holds
              const uint2 b = *reinterpret_cast<const uint2*>(br + i * 8 * bld + 32 * k);
#pragma unroll
              for (int part = 0; part < kParts; ++part) mma_16816<true>(acc[i], f[part], b.x, b.y);
            }
          }
          const bool mine = (t < 2 ? j0 : j1) == j;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i][e] = mine ? acc[i][e] : d[i][e];
        }
        if (q * 16 + 4 * t < width) {  // the one place where an output is changed
          uint8_t* w = os + (warp * kLoraTile + g) * kOld + (q * 16 + 4 * t) * kSize;
          if (id0 == a) Four::store(w, 0, Four::add(Four::load(w, 0), d[0][0], d[0][1], d[1][0], d[1][1]));
          w += 8 * kOld;
          if (id1 == a) Four::store(w, 0, Four::add(Four::load(w, 0), d[0][2], d[0][3], d[1][2], d[1][3]));
        }
      }
    }
    if (u + 1 < rows.n) {
      __syncthreads();  // B is replaced
      fetch_b(rows.uniq[u + 1]);
    }
  }
  cp_async_wait<0>();
  __syncthreads();
  const bool copy = p.base != p.out;  // in place, rows without an adapter stay
  uint8_t* out = static_cast<uint8_t*>(p.out) + ((size_t)(t0 + mr) * p.out_ld + o0) * kSize + mc * 16;
  const size_t hop = (size_t)kHop * p.out_ld * kSize;
#pragma unroll
  for (int r = 0; r < kLoraRows; r += kHop)
    if (r + mr < mrows && (copy || rows.ids[r + mr] >= 0))
      *reinterpret_cast<uint4*>(out + r / kHop * hop) = *reinterpret_cast<const uint4*>(os + (r + mr) * kOld + mc * 16);
}

// Units of a decode step at most: one per adapter in use, one more per 16 tokens, tokens without one.
static int lora_units(int tokens, int adapters) {
  const long n = (long)adapters + 1 + tokens / kLoraTile;
  return (int)(n < tokens ? n : tokens);
}
// Inputs per split: whole steps of each warp of a decode step's CTA, whole stages for prompts.
static int lora_per_split(int inputs, int splits, bool group) {
  const int step = group ? 32 * kLoraWarps : kLoraStep;
  return ((inputs + splits - 1) / splits + step - 1) / step * step;
}
// Splits of the inputs, a cluster: for a decode step 1 to 16 CTAs (four an SM at most, one step of its warps each or
// more), for prompts 1 to 8 (one stage each or more).
static int lora_splits(int tokens, int inputs, int ranks, int adapters) {
  const bool group = tokens <= kLoraGroupTokens;
  const long z = group ? 1 : (ranks + 8 * kLoraRankTiles - 1) / (8 * kLoraRankTiles);
  const long base = (group ? lora_units(tokens, adapters) : (tokens + kLoraRows - 1) / kLoraRows) * z;
  const int step = group ? 32 * kLoraWarps : kLoraStep;
  int sp = group ? 16 : 8;
  while (sp > 1 && (base * sp > 4 * 148 || inputs < sp * step)) sp /= 2;
  return sp;
}

template <bool OB, int kBlocks, int kFetch>
static int run_lora_group(const LoraArgs& p, cudaStream_t st) {
  static_assert(lora_group_smem(kLoraMaxRanks, 3) <= 45 * 1024, "no raised limit needed");
  static std::atomic<uint64_t> wide_set{0};  // devices on which clusters of more than 8 are allowed
  auto kern = lora_group_kernel<OB, kBlocks, kFetch>;
  int rc = ensure_attribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1, wide_set);
  if (rc) return rc;
  return launch_cluster(kern, dim3(p.splits, lora_units(p.tokens, p.adapters)), dim3(kLoraWarps * 32),
                        lora_group_smem(p.rank * p.slices, OB ? 2 : 3), st, p.splits, p);
}

template <bool OB>
static int run_lora_prompt(const LoraArgs& p, cudaStream_t st) {
  const int R = p.rank * p.slices;
  const unsigned tiles = (p.tokens + kLoraRows - 1) / kLoraRows, z = (R + 8 * kLoraRankTiles - 1) / (8 * kLoraRankTiles);
  constexpr size_t ring = (size_t)kLoraStages * kLoraStageBytes;
  static_assert(ring >= (size_t)kLoraRows * (kLoraRankTiles * 8 + 4) * 4, "the sums take the ring's place");
  static std::atomic<uint64_t> shrink_set{0}, expand_set[4];  // per kernel: devices with the limit raised
  int rc = ensure_smem_limit(lora_shrink_kernel, ring, shrink_set);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles, p.splits, z);
  cfg.blockDim = dim3(kLoraWarps * 32);
  cfg.dynamicSmemBytes = ring;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = p.splits;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, lora_shrink_kernel, p) != cudaSuccess) return CCUT_ERR_CUDA;
  auto smem = [](size_t R, size_t rank) {
    const bool regs = rank == 16 || rank == 32 || rank == 64;
    return (regs ? 0 : (size_t)(OB ? 2 : 3) * kLoraRows * lora_ld((int)R) * 2) + kLoraOutputs * lora_ld((int)rank) * 2 +
           kLoraRows * (kLoraOutputs + 16) * (OB ? 2 : 4);
  };
  auto kern = p.rank == 16   ? lora_expand_kernel<1, OB>
              : p.rank == 32 ? lora_expand_kernel<2, OB>
              : p.rank == 64 ? lora_expand_kernel<4, OB>
                             : lora_expand_kernel<0, OB>;
  rc = ensure_smem_limit(kern, smem(kLoraMaxRanks, kLoraMaxRanks),
                         expand_set[p.rank == 16 ? 0 : p.rank == 32 ? 1 : p.rank == 64 ? 2 : 3]);
  if (rc) return rc;
  // begun while the shrink kernel runs, whatever the call's size: that was launched without the attribute, so all that
  // is read before the wait is complete
  const bool on = g_pdl_on;
  g_pdl_on = pdl_enabled();
  rc = launch_k(kern, dim3(tiles, (p.outputs + kLoraOutputs - 1) / kLoraOutputs), dim3(kLoraWarps * 32),
                smem(R, p.rank), st, p);
  g_pdl_on = on;
  return rc;
}

}  // namespace ccut

using namespace ccut;

extern "C" {

size_t ccut_lora_workspace_bytes(int tokens, int inputs, int rank, int slices, int adapters) {
  if (tokens < 0 || inputs <= 0 || rank <= 0 || slices <= 0 || adapters < 0 || (long)rank * slices > kLoraMaxRanks)
    return 0;
  return tokens <= kLoraGroupTokens ? 0 : 256 + (size_t)tokens * rank * slices * sizeof(float);
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
  const size_t need = ccut_lora_workspace_bytes(tokens, inputs, rank, slices, adapters);
  if (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || ws_bytes < need)) return CCUT_ERR_WORKSPACE;
  const int R = rank * slices;
  p.x = x, p.a = a, p.b = b, p.scales = scales, p.ids = ids;
  p.tokens = tokens, p.inputs = inputs, p.outputs = (int)o, p.rank = rank, p.slices = slices, p.adapters = adapters;
  p.base = base, p.base_ld = base_ld, p.out = out, p.out_ld = out_ld;
  if (need > 0) p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 256);
  p.splits = lora_splits(tokens, inputs, R, adapters);
  p.k_per_split = lora_per_split(inputs, p.splits, tokens <= kLoraGroupTokens);
  if ((o + kLoraOutputs - 1) / kLoraOutputs > 65535) return CCUT_ERR_UNSUPPORTED;
  const bool ob = dtype == CCUT_OUT_BF16;
  if (tokens <= kLoraGroupTokens) {
    // what a warp has on its way: more outputs at ranks of up to 32, more of B's k steps above (64 tokens, rank 3 x 64,
    // 4096 inputs, 6144 outputs: 21.2 us, 21.9 with the other).  As many blocks as three CTAs an SM have registers for
    // (8 spill: 12.3 us at 5120 outputs); between 2 and 6 it matters little: 5120 outputs 10.2 us with 5, 10.6 to 10.9
    // with the others, 2560 9.2 (9.1 to 9.5), 2048 8.3 (8.0 to 8.5), 8192 of 4096 inputs 12.7 (12.5 to 12.9)
    if (rank <= 32) return ob ? run_lora_group<true, 5, 2>(p, stream) : run_lora_group<false, 5, 2>(p, stream);
    return ob ? run_lora_group<true, 3, 4>(p, stream) : run_lora_group<false, 3, 4>(p, stream);
  }
  return ob ? run_lora_prompt<true>(p, stream) : run_lora_prompt<false>(p, stream);
}

}  // extern "C"
