// kv4_attn.cu -- grouped-query attention over the 4-bit kv cache (format: kv4.cuh); long query blocks:
// kv4_prefill.cu.
//
// q bf16 [batch, heads, seq, d]; batch row b reads slot slots[b], its query i sees positions
// <= starts[b] + i (and < kv_len); query head h reads kv head h / (heads / kv_heads).
//   x_j = scale * sum_d q_d (s_jg c_jd + m_jg), optionally soft-capped; o = sum_j softmax(x)_j v^_j
//
// Short query blocks (decode steps; kv4_attn_kernel).  Bound: HBM, 36 bytes per 64 features of k and v
// once per kv head; what stands in the way of that is the instructions that turn nibbles into MMA
// operands, so the kernel is built around needing few of them:
// - No dequantization.  A nibble masked in place is an fp16 subnormal: bits 0-3 hold c 2^-24, bits
//   4-7 hold c 2^-20 (16 times as much).  One AND makes an operand pair, exact; the powers of two go
//   into q (odd features divided by 16) and into the output.  The MMA multiplies the codes, and the
//   group's scale and minimum are applied to the products:
//   x = sum_g s_g (q_g . c_g) + m_g (sum q_g),  o = sum_j (p_j s_jg) c_j + (sum_j p_j m_jg),
//   the minima of k by one more MMA (their fp16 pairs times sum q_g in two fp16 parts).
// - Positions are the M of m16n8k16, the query rows of a kv head the N: 8 rows take half the MMAs
//   they would take as the M.  The order of the k index is free, so a lane's operands are the next
//   bytes of a cache row (no ldmatrix), and the scores' accumulators become the second product's operand
//   by movmatrix.
// - Each warp streams its own tiles through a cp.async ring, with no barrier between warps: up to 8 query rows
//   (one n-tile) tiles of 32 positions, three deep, with more rows (two n-tiles) 16 positions, four deep.
//   32-byte units are placed so that the reads of both operands touch every bank once.
//   (Prefetching into registers instead took 168 of them and left three CTAs an SM.)
// - The running maximum moves only when a score passes it by 2^4 (one vote a tile instead of
//   six shuffles a row pair): probabilities stay below 2^4, and fp16's range has room for that (kKv4Room).
// - Tiles that every row sees in whole run without mask tests; the few others (the last tile, the diagonal
//   of a query block) run a masked copy.
// - Work is cut evenly whatever the lengths: the blocks of 128 (8 rows) or 64 positions of all (sequence, tile of
//   query rows, kv head) units form one line (a call of up to kKv4Uncut positions has one block a unit), found from
//   starts on the device, and each CTA of one resident round takes an equal span of it.  A unit inside one span is finished there; of the others a span
//   leaves at most two partial results (the first and the last of its units), which a second kernel joins.
//   Equal chunks per sequence cost a prologue, a reduction and a partial result every chunk instead (one
//   sequence of 131071 positions, when this was changed: 54 us in chunks, 22 in spans).
// Measured (8 query heads per kv head, d = 128): 64 sequences of 3001..8191 positions 50 us, 4.1 TB/s of codes
// and params (0.64 of a copy's rate); the schedulers issue in 0.55 of the cycles, three warps each in chains of
// dependent instructions (four, at 128 registers: 53 us).  One sequence of 131071: 13 us in two launches.
// One of 513: 8.5 us, latency.
// Roundings to fp16: q, scaled to its row's largest element (2^-35 of it is kept), and sum q_g (2^-15
// of the largest element); p s_v, scaled by the row's power of two R that brings the largest v scale it has
// seen to [2^10, 2^11) (11 bits, and 2^-35 of that scale absolutely; with fp32 output a second fp16 part
// keeps 22 bits, and 2^-35).  Everything else, running maximum, sums and outputs, is fp32; the leading zeros
// of subnormal operands are bits that the tensor cores' sums do without, which with fp32 output shows as 1e-6
// of the largest value (decode of 513 to 131071 positions), 1.5e-5 to 2.8e-4 of the output's norm.
// The codes are not centred, so the sums of p s c and of p m cancel and the rounding of p s_v counts two to three
// times: 64 ragged caches' bf16 outputs are 1.74e-3 off (relative norm), where the rounding to bf16 alone makes 1.66e-3.
// What it would cost: two parts 56 us for 50 (1.66e-3); codes centred at 7.5 by the sum of the rounded p s_v, one
// more product, 52.6 us (1.67e-3).
#include <math.h>

#include "kv4.cuh"

namespace ccut {

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
  int batch, row_tiles;  // row_tiles: tiles of 8 or 16 query rows per kv head
  int ctas;              // grid of the attention kernel
  int block;             // positions per block of work, a multiple of kKv4Block
  float2* ml;            // [ctas][2][rows of a tile] running maximum (log2 units) and sum of a partial unit
  float* acc;            // [ctas][2][rows of a tile][d] its unnormalised output
};

constexpr int kKv4Warps = 4;
// Positions per warp step: 32 with one n-tile (two independent chains of MMAs and one vote a step), 16 with two
// (the registers hold no more).
template <int NT>
constexpr int kKv4Tile = NT == 1 ? 32 : 16;
template <int NT>
constexpr int kKv4Block = kKv4Warps * kKv4Tile<NT>;  // positions per block of work

constexpr float kLog2e = 1.4426950408889634f;

CCUT_DEVICE uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
CCUT_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CCUT_DEVICE uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
CCUT_DEVICE __half2 as_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
CCUT_DEVICE float2 unpack_f16(uint32_t u) { return __half22float2(as_half2(u)); }
CCUT_DEVICE float low_f16(uint32_t u) { return __low2float(as_half2(u)); }
CCUT_DEVICE float high_f16(uint32_t u) { return __high2float(as_half2(u)); }
CCUT_DEVICE float pow2f(int e) { return __int_as_float((e + 127) << 23); }
CCUT_DEVICE int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 255) - 127; }

// A warp's tile in shared memory: k codes, v codes (32-byte units, see the placements), then the (scale,
// minimum) pairs of k and of v.
template <int D, int NT>
struct Kv4Stage {
  static constexpr int kCodes = kKv4Tile<NT> * D / 2, kParams = kKv4Tile<NT> * D / 16;
  static constexpr int kBytes = 2 * kCodes + 2 * kParams;
};
template <int NT>
constexpr int kKv4Stages = NT == 1 ? 3 : 4;
template <int D, int NT>
constexpr int kKv4Smem = kKv4Warps * (kKv4Stages<NT> * Kv4Stage<D, NT>::kBytes > 8 * NT * (D + 4) * 4
                                          ? kKv4Stages<NT> * Kv4Stage<D, NT>::kBytes
                                          : 8 * NT * (D + 4) * 4);
// Row i of the MMAs' M (scores) and k (values) index is position kv4_row(i) of its 16: lane t then reads v at
// positions t, t + 4, t + 8, t + 12, four different bank groups for the four t.
CCUT_DEVICE int kv4_row(int i) { return ((i >> 1) & 3) + 4 * (i & 1) + (i & 8); }
// Byte offset of 32-byte unit `gr` (its group) of position r: lanes that read one unit each of positions
// {0, 1, 2, 3}, {4, .., 7} (v) or {0, 4, 1, 5}, {2, 6, 3, 7} (k, half a warp) meet every bank once.
template <int D>
CCUT_DEVICE int kv4_unit(int r, int gr) {
  if constexpr (D == 128) return r * 64 + ((gr ^ (((r >> 1) ^ (r >> 2)) & 1)) * 32);
  else return (r ^ ((r >> 1) & 2)) * 32;
}
// cp.async of N (16, 8 or 4) bytes to shared address `to`; kChecked: zeros when !in
template <int N, bool kChecked>
CCUT_DEVICE void copy_in(uint32_t to, const uint8_t* from, bool in) {
  if constexpr (N == 16) {
    if constexpr (kChecked)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
    else
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  } else {
    if constexpr (kChecked)
      asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(to), "l"(from), "r"(in ? N : 0), "n"(N)
                   : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(N) : "memory");
  }
}

// Four features of an output row.
template <bool OUT_BF16>
CCUT_DEVICE void kv4_store(void* out, long long at, const float4& v) {
  if constexpr (OUT_BF16) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  } else {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = v;
  }
}

// The line of work: sequence b has kv4_blocks blocks of positions in each of its units, at least one (a
// unit that sees nothing still writes its zeros).
CCUT_DEVICE int kv4_seen(const Kv4AttnArgs& a, int b) {  // positions its last query sees
  const int slot = a.slots[b], start = a.starts[b];
  return slot >= 0 && slot < a.num_slots && start >= 0 ? min(a.kv_len, min(start, a.kv_len) + a.seq) : 0;
}
CCUT_DEVICE int kv4_blocks(const Kv4AttnArgs& a, int seen) { return max(1, (seen + a.block - 1) / a.block); }
// Whole warp.  Length of the line.  `mine`: blocks of sequence `lane`, for kv4_find.
CCUT_DEVICE int kv4_total(const Kv4AttnArgs& a, int lane, int& mine) {
  mine = lane < a.batch ? kv4_blocks(a, kv4_seen(a, lane)) : 0;
  unsigned n = mine;  // no overflow: the line is bounded at launch
  for (int b = lane + 32; b < a.batch; b += 32) n += kv4_blocks(a, kv4_seen(a, b));
  return (int)__reduce_add_sync(0xffffffffu, n) * a.kv_heads * a.row_tiles;
}
// Whole warp.  The sequence at place `at` of the line, and the place of its first block.
CCUT_DEVICE int kv4_find(const Kv4AttnArgs& a, int lane, int mine, int at, int& first) {
  const int units = a.kv_heads * a.row_tiles;
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int n = b0 == 0 ? mine : b0 + lane < a.batch ? kv4_blocks(a, kv4_seen(a, b0 + lane)) : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, base + sum * units > at);
    if (past) {
      const int w = __ffs(past) - 1;
      first = base + __shfl_sync(0xffffffffu, sum - n, w) * units;
      return b0 + w;
    }
    base += __shfl_sync(0xffffffffu, sum, 31) * units;
  }
  first = base;
  return a.batch;  // not reached for places on the line
}
// The line in n spans, the first total % n of them one longer: where span i begins, and the span of a place.
CCUT_DEVICE int kv4_span(int total, int n, int i) { return i * (total / n) + min(i, total % n); }
CCUT_DEVICE int kv4_span_of(int total, int n, int at) {
  const int per = total / n, cut = (total % n) * (per + 1);
  return at < cut ? at / (per + 1) : total % n + (at - cut) / per;
}

template <int D, int NT>
constexpr int kKv4Resident = D == 64 ? (NT == 1 ? 5 : 4) : (NT == 1 ? 3 : 2);  // CTAs per SM, by registers

template <int D, int NT, bool OUT_BF16>
__global__ void __launch_bounds__(kKv4Warps * 32, kKv4Resident<D, NT>) kv4_attn_kernel(Kv4AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int G = D / kKv4Group;
  constexpr int kRows = 8 * NT;
  constexpr uint32_t M0 = 0x000F000Fu, M1 = 0x00F000F0u;
  using St = Kv4Stage<D, NT>;
  constexpr int kTile = kKv4Tile<NT>, kBlock = kKv4Block<NT>, kStages = kKv4Stages<NT>, U = kTile / 16;
  extern __shared__ __align__(16) uint8_t smem[];  // the rings, then the warps' outputs
  float(*sm_o)[kRows][D + 4] = reinterpret_cast<float(*)[kRows][D + 4]>(smem);
  __shared__ float sm_m[kKv4Warps][kRows], sm_l[kKv4Warps][kRows], sm_f[kKv4Warps][kRows];
  __shared__ long long sm_at[kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int grp = a.heads / a.kv_heads, nrows = grp * a.seq;
  int mine, first;
  const int total = kv4_total(a, lane, mine), spans = min(a.ctas, total);
  if ((int)blockIdx.x >= spans) return;
  const int begin = kv4_span(total, spans, blockIdx.x), end = kv4_span(total, spans, blockIdx.x + 1);
  int b = kv4_find(a, lane, mine, begin, first);
  int at = begin;

  while (at < end) {
  const int seen = kv4_seen(a, b), nblocks = kv4_blocks(a, seen);
  const int unit = (at - first) / nblocks, block0 = (at - first) % nblocks;
  const int block1 = min(nblocks, block0 + (end - at));
  const bool whole_unit = block0 == 0 && block1 == nblocks;
  const int part = blockIdx.x * 2 + (at != begin);
  const int kvh = unit % a.kv_heads, r0 = unit / a.kv_heads * kRows;
  const int start = min(a.starts[b], a.kv_len);
  const int last_row = min(nrows, r0 + kRows) - 1;
  const int k0 = block0 * a.block;
  // positions any row of this tile sees in this segment
  const int k1 = seen > 0 ? min(min(seen, block1 * a.block), start + last_row / grp + 1) : 0;
  const size_t row_base = seen > 0 ? (size_t)a.slots[b] * (size_t)a.slot_rows + (size_t)kvh * a.max_len : 0;

  // ---- the query rows as B fragments (row n = g of n-tile nt; features t * 16 .. of each group) ----
  uint32_t qf[NT][G][4][2], qm[NT];  // qm: sum q_g of the groups, high parts in lanes t = 0, the rest in t = 1
  float fr[NT][2];                   // columns 2t, 2t + 1: factor of the products
  int lim[NT][2];                    // last visible position
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + nt * 8 + g;
    float x[G][16], mx = 0.f, sum[G];
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      uint4 u[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (r < nrows) {
        const uint16_t* p =
            a.q + (((size_t)b * a.heads + kvh * grp + r % grp) * a.seq + r / grp) * D + gr * kKv4Group + t * 16;
        u[0] = reinterpret_cast<const uint4*>(p)[0];
        u[1] = reinterpret_cast<const uint4*>(p)[1];
      }
      const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
      sum[gr] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[gr][2 * i] = __uint_as_float(w[i] << 16);
        x[gr][2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        sum[gr] += x[gr][2 * i] + x[gr][2 * i + 1];
        mx = fmaxf(mx, fmaxf(fabsf(x[gr][2 * i]), fabsf(x[gr][2 * i + 1])));
      }
      sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
      sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int e = min(max(exponent_of(mx), -90), 90);  // |q| 2^-e in [1, 2)
    const float f = pow2f(14 - e);                     // the operand in [2^14, 2^15)
#pragma unroll
    for (int gr = 0; gr < G; ++gr)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // features d0 + {2h, 2h + 4} and {2h + 1, 2h + 5}, the latter / 16
          const float* d = &x[gr][w * 8 + 2 * h];
          qf[nt][gr][w * 2 + h][0] = pack_f16(d[0] * f, d[4] * f);
          qf[nt][gr][w * 2 + h][1] = pack_f16(d[1] * (f * 0.0625f), d[5] * (f * 0.0625f));
        }
    // operand pair of the minima: (m of group 0, of group 1), or with one group the row's (s, m)
    const float s0 = G == 2 ? sum[0] * pow2f(-10 - e) : 0.f, s1 = sum[G - 1] * pow2f(-10 - e);
    const uint32_t hi = pack_f16(s0, s1);
    const float2 hf = unpack_f16(hi);
    qm[nt] = t == 0 ? hi : t == 1 ? pack_f16(s0 - hf.x, s1 - hf.y) : 0u;
    const float back = pow2f(10 + e) * (a.scale * kLog2e);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      fr[nt][c] = __shfl_sync(0xffffffffu, back, (2 * t + c) * 4);  // a lane that holds row 2t + c
      lim[nt][c] = start + (r0 + nt * 8 + 2 * t + c) / grp;
    }
  }

  float m[NT][2], l[NT][2], am[NT][G][2], o[NT][D / 16][4], R[NT][2];
  __half r_inv = __ushort_as_half(0);  // the least scale that needs a smaller R; 0 before the first tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[nt][c] = -INFINITY, l[nt][c] = 0.f, R[nt][c] = pow2f(30 + kKv4Room);  // 2^-30: below every scale
#pragma unroll
      for (int gr = 0; gr < G; ++gr) am[nt][gr][c] = 0.f;
    }
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
  }

  // This lane's part of a tile: 16-byte chunks lane, lane + 32, .. of the codes, and a position's pair(s):
  // with 32 positions of k and then of v, with 16 of k (lanes 0-15) or of v.  The addresses move from
  // one tile of the warp to its next; positions at or past k1 come as zeros.
  const uint8_t* ring = smem + warp * kStages * St::kBytes;
  constexpr int kPer = D / 32, kStepRows = 32 / kPer;  // chunks per position, positions per 32 chunks
  const int cr = lane / kPer, first_tile = k0 + warp * kTile, prow = U == 2 ? lane : lane & 15;
  const uint32_t to_codes = smem_u32(ring) + kv4_unit<D>(cr, lane % kPer >> 1) + (lane & 1) * 16;
  const uint32_t to_params = smem_u32(ring) + 2 * St::kCodes + lane * (D / 16);
  const uint8_t* kc = a.kc + (row_base + first_tile) * (D / 2) + lane * 16;
  const uint8_t* vc = a.vc + (row_base + first_tile) * (D / 2) + lane * 16;
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(U == 2 || lane < 16 ? a.kp : a.vp) + (row_base + first_tile + prow) * (D / 16);
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.vp) + (row_base + first_tile + prow) * (D / 16);  // U == 2
  auto copy_tile = [&](uint32_t stage, int left, auto checked) {
    constexpr bool kC = decltype(checked)::value;  // a position past the end is not touched, nor is its address formed
#pragma unroll
    for (int i = 0; i < St::kCodes / 512; ++i) {
      const bool in = cr + kStepRows * i < left;
      copy_in<16, kC>(to_codes + stage + i * 512, kC && !in ? a.kc : kc + i * 512, in);
      copy_in<16, kC>(to_codes + stage + St::kCodes + i * 512, kC && !in ? a.vc : vc + i * 512, in);
    }
    const bool in = prow < left;
    copy_in<D / 16, kC>(to_params + stage, kC && !in ? reinterpret_cast<const uint8_t*>(a.kp) : kp, in);
    if constexpr (U == 2)
      copy_in<D / 16, kC>(to_params + stage + St::kParams, kC && !in ? reinterpret_cast<const uint8_t*>(a.vp) : vp, in);
    kc += kBlock * (D / 2);
    vc += kBlock * (D / 2);
    kp += kBlock * (D / 16);
    if constexpr (U == 2) vp += kBlock * (D / 16);
  };
  auto issue = [&](int tile, int stage) {
    const int left = k1 - k0 - tile * kTile;
    if (left >= kTile) copy_tile(stage * St::kBytes, left, std::false_type{});
    else copy_tile(stage * St::kBytes, left, std::true_type{});
  };
  const int kr = kv4_row(g);                          // this lane's score rows: positions kr and kr + 8
  const int k_unit[2] = {kv4_unit<D>(kr, 0) + t * 8, kv4_unit<D>(kr, 1) + t * 8};
  const int v_unit[2][2] = {{kv4_unit<D>(t, 0) + g * 4, kv4_unit<D>(t, 1) + g * 4},
                            {kv4_unit<D>(t + 4, 0) + g * 4, kv4_unit<D>(t + 4, 1) + g * 4}};

  auto step = [&](const uint8_t* st, int p0, auto masked_tag) {
    constexpr bool kMasked = decltype(masked_tag)::value;
    float sc[U][NT][4];  // element i: row g + 8 (i >> 1), column 2t + (i & 1)
    bool vis[U][NT][4];
    uint32_t vpw[U][2][G];
    bool need = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t kpw[2][G];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint8_t* p = st + 2 * St::kCodes + (16 * u + 8 * h + kr) * (D / 16);
        if constexpr (G == 2) {
          const uint2 uk = *reinterpret_cast<const uint2*>(p), uv = *reinterpret_cast<const uint2*>(p + St::kParams);
          kpw[h][0] = uk.x, kpw[h][G - 1] = uk.y, vpw[u][h][0] = uv.x, vpw[u][h][G - 1] = uv.y;
        } else {
          kpw[h][0] = *reinterpret_cast<const uint32_t*>(p);
          vpw[u][h][0] = *reinterpret_cast<const uint32_t*>(p + St::kParams);
        }
      }
      const uint32_t fm[4] = {G == 2 ? __byte_perm(kpw[0][0], kpw[0][G - 1], 0x7632) : kpw[0][0],
                              G == 2 ? __byte_perm(kpw[1][0], kpw[1][G - 1], 0x7632) : kpw[1][0], 0u, 0u};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[u][nt][i] = 0.f;
        mma_16816<false>(sc[u][nt], fm, qm[nt], 0u);
      }
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        float c4[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) c4[nt][i] = 0.f;
        const uint2 ka = *reinterpret_cast<const uint2*>(st + k_unit[gr] + u * 16 * (D / 2));
        const uint2 kb = *reinterpret_cast<const uint2*>(st + k_unit[gr] + (u * 16 + 8) * (D / 2));
        const uint32_t w0[2] = {ka.x, ka.y}, w1[2] = {kb.x, kb.y};
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t u0 = w0[w] >> (8 * h), u1 = w1[w] >> (8 * h);
            const uint32_t f[4] = {u0 & M0, u1 & M0, u0 & M1, u1 & M1};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma_16816<false>(c4[nt], f, qf[nt][gr][w * 2 + h][0], qf[nt][gr][w * 2 + h][1]);
          }
        const float s[2] = {low_f16(kpw[0][gr]), low_f16(kpw[1][gr])};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[u][nt][i] = fmaf(s[i >> 1], c4[nt][i], sc[u][nt][i]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& x = sc[u][nt][i];
          x *= fr[nt][i & 1];
          if (a.softcap > 0.f) x = tanhf(x * (1.f / kLog2e) / a.softcap) * (a.softcap * kLog2e);
          if constexpr (kMasked) {
            const int p = p0 + 16 * u + kr + 8 * (i >> 1);
            vis[u][nt][i] = p < k1 && p <= lim[nt][i & 1];
            if (!vis[u][nt][i]) x = -INFINITY;
          }
          need |= x > m[nt][i & 1] + kKv4Lag;
        }
    }
    __half2 top = __hmax2(as_half2(vpw[0][0][0]), as_half2(vpw[0][1][0]));
    if constexpr (G == 2) top = __hmax2(top, __hmax2(as_half2(vpw[0][0][G - 1]), as_half2(vpw[0][1][G - 1])));
    if constexpr (U == 2) {
      top = __hmax2(top, __hmax2(as_half2(vpw[U - 1][0][0]), as_half2(vpw[U - 1][1][0])));
      if constexpr (G == 2)
        top = __hmax2(top, __hmax2(as_half2(vpw[U - 1][0][G - 1]), as_half2(vpw[U - 1][1][G - 1])));
    }
    need |= __hge(__low2half(top), r_inv);
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = fmaxf(sc[0][nt][c], sc[0][nt][c + 2]);
          if constexpr (U == 2) v = fmaxf(v, fmaxf(sc[U - 1][nt][c], sc[U - 1][nt][c + 2]));
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
          v = v > m[nt][c] + kKv4Lag ? v : m[nt][c];  // by the row's own scores: its bits depend on no other row
          const float al = v == m[nt][c] ? 1.f : ex2(m[nt][c] - v);
          m[nt][c] = v;
          l[nt][c] *= al;
#pragma unroll
          for (int gr = 0; gr < G; ++gr) am[nt][gr][c] *= al;
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt) o[nt][mt][c] *= al, o[nt][mt][c + 2] *= al;
        }
      float low = INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = __low2float(top);
          if constexpr (kMasked) {  // of the positions that the row sees
            v = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int gr = 0; gr < G; ++gr) v = fmaxf(v, vis[u][nt][c + 2 * h] ? low_f16(vpw[u][h][gr]) : 0.f);
          }
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
          v = fminf(v, 65504.f);
          if (v * R[nt][c] >= pow2f(kKv4Room)) {
            const float r = pow2f(kKv4Room - 1 - exponent_of(v)), f = r / R[nt][c];
            R[nt][c] = r;
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) o[nt][mt][c] *= f, o[nt][mt][c + 2] *= f;
          }
          low = fminf(low, pow2f(kKv4Room) / R[nt][c]);
        }
      r_inv = __float2half_rn(low);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float p[NT][4], pr[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[nt][i] = ex2(sc[u][nt][i] - m[nt][i & 1]);
          if constexpr (kMasked) p[nt][i] = vis[u][nt][i] ? p[nt][i] : 0.f;  // a row that saw nothing yet has m = -inf
          l[nt][i & 1] += p[nt][i];
          pr[nt][i] = p[nt][i] * R[nt][i & 1];
        }
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        const float sv[2] = {low_f16(vpw[u][0][gr]), low_f16(vpw[u][1][gr])};
        const float mv[2] = {high_f16(vpw[u][0][gr]), high_f16(vpw[u][1][gr])};
        uint32_t wb[NT][2], wl[NT][2];  // p s_v R as the B operand: high part, and the rest
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w[i] = pr[nt][i] * sv[i >> 1];
            if constexpr (kMasked) {  // 0 * NaN stays out
              w[i] = vis[u][nt][i] ? w[i] : 0.f;
              am[nt][gr][i & 1] += vis[u][nt][i] ? p[nt][i] * mv[i >> 1] : 0.f;
            } else {
              am[nt][gr][i & 1] = fmaf(p[nt][i], mv[i >> 1], am[nt][gr][i & 1]);
            }
          }
          const uint32_t h0 = pack_f16(w[0], w[1]), h1 = pack_f16(w[2], w[3]);
          wb[nt][0] = movmatrix_trans(h0);
          wb[nt][1] = movmatrix_trans(h1);
          if constexpr (!OUT_BF16) {
            const float2 b0 = unpack_f16(h0), b1 = unpack_f16(h1);
            wl[nt][0] = movmatrix_trans(pack_f16(w[0] - b0.x, w[1] - b0.y));
            wl[nt][1] = movmatrix_trans(pack_f16(w[2] - b1.x, w[3] - b1.y));
          }
        }
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)  // positions t, t + 4, t + 8, t + 12: k indices 2t, 2t + 1, 2t + 8, 2t + 9
          v[i] = *reinterpret_cast<const uint32_t*>(st + St::kCodes + v_unit[i & 1][gr] +
                                                    (u * 16 + (i >> 1) * 8) * (D / 2));
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x7632 : 0x5410;
          const uint32_t p01 = __byte_perm(v[0], v[1], sel), p23 = __byte_perm(v[2], v[3], sel);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t u0 = p01 >> (8 * h), u1 = p23 >> (8 * h);
            const uint32_t f[4] = {u0 & M0, u0 & M1, u1 & M0, u1 & M1};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816<false>(o[nt][gr * 4 + half * 2 + h], f, wb[nt][0], wb[nt][1]);
              if constexpr (!OUT_BF16) mma_16816<false>(o[nt][gr * 4 + half * 2 + h], f, wl[nt][0], wl[nt][1]);
            }
          }
        }
      }
    }
  };

  // tiles of this warp: warp, warp + 4, ..; the first `whole` of the segment are seen in whole by every row.
  // One commit group per tile (empty past the end), so that wait_group always means "this tile has landed".
  const int ntiles = k1 > k0 ? (k1 - k0 + kTile - 1) / kTile : 0;
  const int whole = k1 > k0 ? max(0, min(k1, start + r0 / grp + 1) - k0) / kTile : 0;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (warp + i * kKv4Warps < ntiles) issue(warp + i * kKv4Warps, i);
    cp_async_commit();
  }
  for (int j = warp, i = 0; j < ntiles; j += kKv4Warps, ++i) {
    cp_async_wait<kStages - 2>();
    __syncwarp();  // every lane's copies of this tile have landed, every lane is done with the tile before
    const int jn = j + (kStages - 1) * kKv4Warps;
    if (jn < ntiles) issue(jn, (i + kStages - 1) % kStages);
    cp_async_commit();
    const uint8_t* st = ring + i % kStages * St::kBytes;
    if (j < whole) step(st, 0, std::false_type{});
    else step(st, k0 + j * kTile, std::true_type{});
  }
  cp_async_wait<0>();
  __syncthreads();  // the warps' outputs take the ring's place

  // ---- join the warps: rows 2t + c of n-tile nt, features 8 g + {0..7} of each group -----------------
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int n = nt * 8 + 2 * t + c;
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) {
        l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], s);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) am[nt][gr][c] += __shfl_xor_sync(0xffffffffu, am[nt][gr][c], s);
      }
      if (g == 0) sm_m[warp][n] = m[nt][c], sm_l[warp][n] = l[nt][c];
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        const float u = pow2f(20) / R[nt][c];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          float* d = &sm_o[warp][n][gr * kKv4Group + g * 8 + mt * 2];
          d[0] = fmaf(o[nt][gr * 4 + mt][c], 16.f * u, am[nt][gr][c]);
          d[1] = fmaf(o[nt][gr * 4 + mt][c + 2], u, am[nt][gr][c]);
        }
      }
    }
  __syncthreads();
  if (threadIdx.x < kRows) {  // each warp's factor for row n, and where the row goes (-1: past the last)
    const int n = threadIdx.x, r = r0 + n;
    float M = -INFINITY, L = 0.f, f[kKv4Warps];
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) M = fmaxf(M, sm_m[w][n]);
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) {
      f[w] = ex2(sm_m[w][n] - (M == -INFINITY ? 0.f : M));  // 0 for a warp that saw nothing
      L = fmaf(sm_l[w][n], f[w], L);
    }
    if (!whole_unit) a.ml[part * kRows + n] = make_float2(M, L);
    const float inv = !whole_unit ? 1.f : L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) sm_f[w][n] = f[w] * inv;
    sm_at[n] = r >= nrows    ? -1
               : !whole_unit ? (long long)part * kRows + n
                             : ((long long)b * a.heads + kvh * grp + r % grp) * a.seq + r / grp;
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < kRows * D / 4; idx += kKv4Warps * 32) {
    const int n = idx / (D / 4), d = idx % (D / 4) * 4;
    const long long row = sm_at[n];
    if (row < 0) continue;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) {
      const float f = sm_f[w][n];
      const float4 x = *reinterpret_cast<const float4*>(&sm_o[w][n][d]);
      v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
    }
    if (!whole_unit) *reinterpret_cast<float4*>(a.acc + row * D + d) = v;
    else kv4_store<OUT_BF16>(a.out, row * D + d, v);
  }
  at += block1 - block0;
  if (at < end) {
    if (at >= first + nblocks * a.kv_heads * a.row_tiles) {
      first = at;
      ++b;
    }
    __syncthreads();  // the join's shared memory is used again
  }
  }
}

// Joins the partial results of a query row (none: the row was finished by its span).  W warps a row, at least
// eight a CTA: warp w of a row takes spans w, w + W, .. of the row's unit, each lane D / 32 features; the W
// sums are added in warp order.  The line is looked up before the wait for the attention kernel: slots and
// starts were there before that began.
template <int D, int NT, int W, bool OUT_BF16>
__global__ void __launch_bounds__(W > 8 ? W * 32 : 256) kv4_merge_kernel(Kv4AttnArgs a, long long rows) {
  constexpr int E = D / 32, kRows = 8 * NT, kPer = W > 8 ? 1 : 8 / W;
  __shared__ float so[W][D];
  __shared__ float2 sl[W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp % W;
  const long long row = (long long)blockIdx.x * kPer + warp / W;
  const bool live = row < rows;
  int b = 0, h = 0, i = 0;
  if (live) i = (int)(row % a.seq), b = (int)(row / a.seq / a.heads), h = (int)(row / a.seq % a.heads);
  const int grp = a.heads / a.kv_heads, r = i * grp + h % grp;
  unsigned all = 0, before = 0;
  for (int j = lane; j < a.batch; j += 32) {
    const int n = kv4_blocks(a, kv4_seen(a, j));
    all += n;
    before += j < b ? n : 0;
  }
  const int units = a.kv_heads * a.row_tiles;
  const int total = (int)__reduce_add_sync(0xffffffffu, all) * units;
  const int nblocks = kv4_blocks(a, kv4_seen(a, b));
  const int first = (int)__reduce_add_sync(0xffffffffu, before) * units + (r / kRows * a.kv_heads + h / grp) * nblocks;
  const int spans = min(a.ctas, total);
  const int c0 = kv4_span_of(total, spans, first), c1 = kv4_span_of(total, spans, first + nblocks - 1);
  // in span c0 the unit comes after others (partial result 1) unless it begins the span; in the rest it begins it
  const int late = kv4_span(total, spans, c0) < first ? 1 : 0;
  pdl_wait();
  pdl_trigger();
  if (!live || c0 == c1) return;  // the same for every warp of a row; with one row a CTA for the whole CTA
  // one pass with a running maximum: no load waits for another
  float M = -INFINITY, L = 0.f, v[E] = {};
  auto take = [&](float m2, float l2, const float(&x)[E]) {
    const float top = fmaxf(M, m2), base = top == -INFINITY ? 0.f : top;
    const float f = ex2(M - base), f2 = ex2(m2 - base);
    M = top;
    L = fmaf(L, f, l2 * f2);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = fmaf(v[e], f, x[e] * f2);
  };
#pragma unroll 8
  for (int c = c0 + w; c <= c1; c += W) {
    const size_t part = (size_t)(2 * c + (c == c0 ? late : 0)) * kRows + r % kRows;
    const float2 ml = a.ml[part];
    const float* p = a.acc + part * D + lane * E;
    float x[E];
    if constexpr (E == 4) {
      const float4 y = *reinterpret_cast<const float4*>(p);
      x[0] = y.x, x[1] = y.y, x[E - 2] = y.z, x[E - 1] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(p);
      x[0] = y.x, x[1] = y.y;
    }
    take(ml.x, ml.y, x);
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) so[warp][lane * E + e] = v[e];
    if (lane == 0) sl[warp] = make_float2(M, L);
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int x = 1; x < W; ++x) {
      float y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = so[x][lane * E + e];
      take(sl[x].x, sl[x].y, y);
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float y = v[e] * inv;
    if constexpr (OUT_BF16) static_cast<__nv_bfloat16*>(a.out)[row * D + lane * E + e] = __float2bfloat16_rn(y);
    else static_cast<float*>(a.out)[row * D + lane * E + e] = y;
  }
}

// Query rows per tile: 8 where a kv head has no more, else 16.
static int kv4_rows(int heads, int kv_heads, int seq) { return (long)(heads / kv_heads) * seq <= 8 ? 8 : 16; }
// Positions per block of work: a step of every warp, or all positions where they are few, so that no unit is
// cut and nothing is left to join: 64 sequences of up to 1000 17.6 us uncut, 19.5 cut; 8 of up to 690 9.5 and
// 9.4.  The limit looks at the positions alone, for calls from the host: one sequence of 1024 takes 11.0 us uncut and
// 7.7 cut, but the second launch costs the host 5 us of a call's 20.  A captured graph pays the 3 us.
constexpr int kKv4Uncut = 1024;
static int kv4_block(int rows, int kv_len) {
  const int step = rows == 8 ? kKv4Block<1> : kKv4Block<2>;
  return kv_len <= kKv4Uncut ? (kv_len > 0 ? (kv_len + step - 1) / step * step : step) : step;
}
static long long kv4_row_tiles(int heads, int kv_heads, int seq) {
  const long long rows = (long long)(heads / kv_heads) * seq, per = kv4_rows(heads, kv_heads, seq);
  return (rows + per - 1) / per;
}
// One resident round, or one block each where there are fewer; a unit in at most about kKv4Parts parts, whose
// joining would else take longer than the shorter spans save.
constexpr int kKv4Parts = 128;
static int kv4_ctas(int batch, int heads, int kv_heads, int seq, int kv_len, int head_dim) {
  const bool one = kv4_rows(heads, kv_heads, seq) == 8;
  const int most = 148 * (head_dim == 64 ? (one ? kKv4Resident<64, 1> : kKv4Resident<64, 2>)
                                         : (one ? kKv4Resident<128, 1> : kKv4Resident<128, 2>));
  const int block = kv4_block(one ? 8 : 16, kv_len);
  const long long blocks = kv_len > 0 ? (kv_len + block - 1) / block : 1;
  const long long n = kv4_row_tiles(heads, kv_heads, seq) * kv_heads * batch;
  const long long ctas = n * (blocks < kKv4Parts ? blocks : kKv4Parts);
  return n >= most || ctas >= most ? most : (int)ctas;
}

template <int D, int NT, bool OB>
static int run_kv4_attention(const Kv4AttnArgs& a, cudaStream_t st) {
  static std::atomic<uint64_t> smem_set{0};  // devices with the limit raised
  int rc = ensure_smem_limit(kv4_attn_kernel<D, NT, OB>, kKv4Smem<D, NT>, smem_set);
  if (rc) return rc;
  rc = launch_k(kv4_attn_kernel<D, NT, OB>, dim3(a.ctas), dim3(kKv4Warps * 32), kKv4Smem<D, NT>, st, a);
  if (rc || a.kv_len <= a.block) return rc;  // one block a unit: no unit is cut
  // a warp per row where few spans share a unit, else a CTA
  const long long rows = (long long)a.batch * a.heads * a.seq, units = (long long)a.batch * a.kv_heads * a.row_tiles;
  if (a.ctas <= 8 * units)
    return launch_k(kv4_merge_kernel<D, NT, 1, OB>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, a, rows);
  return launch_k(kv4_merge_kernel<D, NT, 16, OB>, dim3((unsigned)rows), dim3(512), 0, st, a, rows);
}

}  // namespace ccut

using namespace ccut;

extern "C" {

size_t ccut_kv4_attention_workspace_bytes(int batch, int heads, int kv_heads, int seq, int kv_len, int head_dim) {
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq < 0 || kv_len < 0 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  if (batch > 0 && seq > 0 && kv4_prefill_fits(batch, heads, kv_heads, seq, kv_len))
    return kv4_prefill_workspace(batch, heads, kv_heads, seq, kv_len, head_dim);
  if (batch == 0 || seq == 0 || kv_len <= kv4_block(kv4_rows(heads, kv_heads, seq), kv_len)) return 256;
  return 256 + (size_t)kv4_ctas(batch, heads, kv_heads, seq, kv_len, head_dim) * 2 * kv4_rows(heads, kv_heads, seq) *
                   (head_dim + 2) * sizeof(float);
}

int ccut_debug_kv4_wait_budget(long long cycles, long long* before) {
  if (cycles < 0 || cycles > kWaitBudgetCycles || !before) return CCUT_ERR_INVALID;
  *before = kv4_wait_budget(cycles);
  return CCUT_OK;
}

int ccut_kv4_attention(const uint16_t* q, const uint8_t* k_codes, const uint16_t* k_params, const uint8_t* v_codes,
                       const uint16_t* v_params, const int32_t* slots, const int32_t* starts, int batch, int heads,
                       int kv_heads, int seq, int head_dim, int max_len, int kv_len, long long slot_rows,
                       int num_slots, float scale, float softcap, void* out, int out_dtype, void* workspace,
                       size_t ws_bytes, ccut_stream_t stream) {
  return ccut_kv4_attention_reported(q, k_codes, k_params, v_codes, v_params, slots, starts, batch, heads, kv_heads, seq,
                                     head_dim, max_len, kv_len, slot_rows, num_slots, scale, softcap, out, out_dtype,
                                     workspace, ws_bytes, nullptr, stream);
}

int ccut_kv4_attention_reported(const uint16_t* q, const uint8_t* k_codes, const uint16_t* k_params,
                                const uint8_t* v_codes, const uint16_t* v_params, const int32_t* slots,
                                const int32_t* starts, int batch, int heads, int kv_heads, int seq, int head_dim,
                                int max_len, int kv_len, long long slot_rows, int num_slots, float scale, float softcap,
                                void* out, int out_dtype, void* workspace, size_t ws_bytes, int32_t* status,
                                ccut_stream_t stream) {
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
      misaligned(v_params, head_dim / 16) || misaligned(out, 16) || misaligned(workspace, 16) || misaligned(status, 4))
    return CCUT_ERR_INVALID;
  // rows in a grid; positions, the line of work in 32 bits (a start past the cache counts as kv_len; blocks round up)
  if ((long long)kv_len + seq > 2147483647LL - 4096) return CCUT_ERR_UNSUPPORTED;
  const double line = (double)batch * kv_heads * kv4_row_tiles(heads, kv_heads, seq) * (kv_len / kKv4Block<2> + 1);
  if ((double)batch * heads * seq > 2147483647.0 || line > 2147483647.0) return CCUT_ERR_UNSUPPORTED;
  const size_t need = ccut_kv4_attention_workspace_bytes(batch, heads, kv_heads, seq, kv_len, head_dim);
  if (need > 256 && (!workspace || ws_bytes < need)) return CCUT_ERR_WORKSPACE;
  if (!(scale > 0.f)) scale = 1.f / sqrtf((float)head_dim);
  if (kv4_prefill_fits(batch, heads, kv_heads, seq, kv_len)) {
    const Kv4Cache c{k_codes, reinterpret_cast<const __half2*>(k_params), v_codes,
                     reinterpret_cast<const __half2*>(v_params), max_len, slot_rows};
    return launch_kv4_prefill(c, q, slots, starts, batch, heads, kv_heads, seq, head_dim, kv_len, num_slots, scale,
                              softcap, out, out_dtype == CCUT_OUT_BF16, workspace, status, stream);
  }
  Kv4AttnArgs a{q, k_codes, reinterpret_cast<const __half2*>(k_params), v_codes,
                reinterpret_cast<const __half2*>(v_params), slots, starts, heads, kv_heads, seq, max_len, kv_len,
                num_slots, slot_rows, scale, softcap, out, batch, (int)kv4_row_tiles(heads, kv_heads, seq),
                kv4_ctas(batch, heads, kv_heads, seq, kv_len, head_dim),
                kv4_block(kv4_rows(heads, kv_heads, seq), kv_len), nullptr, nullptr};
  const int rows = kv4_rows(heads, kv_heads, seq);
  if (need > 256) {
    a.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + 256);
    a.acc = reinterpret_cast<float*>(a.ml + (size_t)a.ctas * 2 * rows);
  }
  const bool ob = out_dtype == CCUT_OUT_BF16, d128 = head_dim == 128;
  if (rows == 8) {
    if (d128) return ob ? run_kv4_attention<128, 1, true>(a, stream) : run_kv4_attention<128, 1, false>(a, stream);
    return ob ? run_kv4_attention<64, 1, true>(a, stream) : run_kv4_attention<64, 1, false>(a, stream);
  }
  if (d128) return ob ? run_kv4_attention<128, 2, true>(a, stream) : run_kv4_attention<128, 2, false>(a, stream);
  return ob ? run_kv4_attention<64, 2, true>(a, stream) : run_kv4_attention<64, 2, false>(a, stream);
}

}  // extern "C"
