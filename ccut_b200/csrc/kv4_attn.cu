// kv4_attn.cu -- grouped-query attention over the 4-bit kv cache (format: kv4.cuh).
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
//   they would take as the M.  The order of the k index is free, so lanes load their operands straight
//   from global memory (8 bytes of 8 rows of k, 4 bytes of 4 rows of v a lane, full 32-byte sectors),
//   no shared memory, and the scores' accumulators become the second product's operand by movmatrix.
// - The running maximum moves only when a score passes it by 2^8 (one vote a tile instead of
//   six shuffles a row pair): probabilities stay below 2^8, and fp16's range has room for that.
// - Tiles that every row sees in whole run without bounds or mask tests, four pointers advancing by
//   constant strides; the few others (the last tile, the diagonal of a query block) run a checked copy.
// Roundings to fp16: q, scaled to its row's largest element (2^-35 of it is kept), and sum q_g (2^-15
// of the largest element); p s_v, scaled by the power of two R that brings the largest v scale seen so
// far to [1/2, 1) (11 bits, and 2^-25 of the largest absolutely; with fp32 output a second fp16 part
// keeps 22).  Everything else, running maximum, sums and outputs, is fp32.
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
  float2* ml;   // [rows][splits] running maximum (log2 units) and sum of a split
  float* acc;   // [rows][splits][d] its unnormalised output
  int chunk, splits;  // positions per split
};

constexpr int kKv4Warps = 4;
constexpr int kKv4Tile = 16;           // positions per warp step

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

// One 16-position tile of a warp as it comes from memory: lane (g, t) holds of k 16 features (8 bytes) per
// group of rows g and g + 8, of v 8 features (4 bytes) per group of rows 2t, 2t + 1, 2t + 8, 2t + 9,
// and the (scale, minimum) pairs of rows g and g + 8.
template <int G>
struct Kv4Tile {
  uint2 k[2][G];
  uint32_t v[4][G];
  uint32_t kp[2][G], vp[2][G];
};

template <int D, int NT, bool OUT_BF16>
__global__ void __launch_bounds__(kKv4Warps * 32) kv4_attn_kernel(Kv4AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int G = D / kKv4Group;
  constexpr int kRows = 8 * NT;
  constexpr uint32_t M0 = 0x000F000Fu, M1 = 0x00F000F0u;
  __shared__ float sm_o[kKv4Warps][kRows][D + 4];
  __shared__ float sm_m[kKv4Warps][kRows], sm_l[kKv4Warps][kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int grp = a.heads / a.kv_heads, nrows = grp * a.seq;
  const int b = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads;
  const int r0 = blockIdx.x * kRows;
  const int slot = a.slots[b];
  int start = min(a.starts[b], a.kv_len);
  const bool valid = slot >= 0 && slot < a.num_slots && start >= 0;
  const int last_row = min(nrows, r0 + kRows) - 1;
  const int k0 = blockIdx.z * a.chunk;
  // positions any row of this CTA sees in this split
  int k1 = valid ? min(min(a.kv_len, k0 + a.chunk), start + last_row / grp + 1) : 0;
  if (a.splits > 1 && k1 <= k0) return;  // the merge kernel does not read a split that sees nothing
  const size_t row_base = valid ? (size_t)slot * (size_t)a.slot_rows + (size_t)kvh * a.max_len : 0;

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

  float m[NT][2], l[NT][2], am[NT][G][2], o[NT][D / 16][4], R = 1.f;
  __half r_inv = __ushort_as_half(0);  // 1 / R; 0 before the first tile
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[nt][c] = -INFINITY, l[nt][c] = 0.f;
#pragma unroll
      for (int gr = 0; gr < G; ++gr) am[nt][gr][c] = 0.f;
    }
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
  }

  // lane addresses at position k0
  const uint8_t* kc = a.kc + (row_base + k0 + g) * (D / 2) + t * 8;
  const uint8_t* vc = a.vc + (row_base + k0 + 2 * t) * (D / 2) + g * 4;
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.kp) + (row_base + k0 + g) * (4 * G);
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.vp) + (row_base + k0 + g) * (4 * G);

  // the tile at the lane addresses; kChecked: `left` positions from its first, the others come as zeros
  auto load = [&](Kv4Tile<G>& x, auto checked, int left) {
    constexpr bool kChecked = decltype(checked)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = !kChecked || g + 8 * h < left;
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
        x.k[h][gr] = in ? __ldg(reinterpret_cast<const uint2*>(kc + h * 8 * (D / 2) + gr * 32)) : make_uint2(0, 0);
      if constexpr (G == 2) {
        const uint2 uk = in ? __ldg(reinterpret_cast<const uint2*>(kp + h * 64)) : make_uint2(0, 0);
        const uint2 uv = in ? __ldg(reinterpret_cast<const uint2*>(vp + h * 64)) : make_uint2(0, 0);
        x.kp[h][0] = uk.x, x.kp[h][G - 1] = uk.y, x.vp[h][0] = uv.x, x.vp[h][G - 1] = uv.y;
      } else {
        x.kp[h][0] = in ? __ldg(reinterpret_cast<const uint32_t*>(kp + h * 32)) : 0u;
        x.vp[h][0] = in ? __ldg(reinterpret_cast<const uint32_t*>(vp + h * 32)) : 0u;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = (i & 1) + 8 * (i >> 1);
      const bool in = !kChecked || 2 * t + p < left;
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
        x.v[i][gr] = in ? __ldg(reinterpret_cast<const uint32_t*>(vc + p * (D / 2) + gr * 32)) : 0u;
    }
  };
  auto advance = [&](int tiles) {
    kc += (long long)tiles * (kKv4Tile * (D / 2));
    vc += (long long)tiles * (kKv4Tile * (D / 2));
    kp += (long long)tiles * (kKv4Tile * 4 * G);
    vp += (long long)tiles * (kKv4Tile * 4 * G);
  };

  auto step = [&](const Kv4Tile<G>& x, int p0, auto masked_tag) {
    constexpr bool kMasked = decltype(masked_tag)::value;
    float sc[NT][4];
    {
      const uint32_t f[4] = {G == 2 ? __byte_perm(x.kp[0][0], x.kp[0][G - 1], 0x7632) : x.kp[0][0],
                             G == 2 ? __byte_perm(x.kp[1][0], x.kp[1][G - 1], 0x7632) : x.kp[1][0], 0u, 0u};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[nt][i] = 0.f;
        mma_16816<false>(sc[nt], f, qm[nt], 0u);
      }
    }
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      float c4[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) c4[nt][i] = 0.f;
      const uint32_t w0[2] = {x.k[0][gr].x, x.k[0][gr].y}, w1[2] = {x.k[1][gr].x, x.k[1][gr].y};
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t u0 = w0[w] >> (8 * h), u1 = w1[w] >> (8 * h);
          const uint32_t f[4] = {u0 & M0, u1 & M0, u0 & M1, u1 & M1};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<false>(c4[nt], f, qf[nt][gr][w * 2 + h][0], qf[nt][gr][w * 2 + h][1]);
        }
      const float s[2] = {low_f16(x.kp[0][gr]), low_f16(x.kp[1][gr])};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[nt][i] = fmaf(s[i >> 1], c4[nt][i], sc[nt][i]);  // row g + 8 (i >> 1), column 2t + (i & 1)
    }
    bool vis[NT][4];
    bool need = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[nt][i] *= fr[nt][i & 1];
        if (a.softcap > 0.f) sc[nt][i] = tanhf(sc[nt][i] * (1.f / kLog2e) / a.softcap) * (a.softcap * kLog2e);
        if constexpr (kMasked) {
          const int p = p0 + g + 8 * (i >> 1);
          vis[nt][i] = p < k1 && p <= lim[nt][i & 1];
          if (!vis[nt][i]) sc[nt][i] = -INFINITY;
        }
        need |= sc[nt][i] > m[nt][i & 1] + 8.f;
      }
    __half2 top = __hmax2(as_half2(x.vp[0][0]), as_half2(x.vp[1][0]));
    if constexpr (G == 2) top = __hmax2(top, __hmax2(as_half2(x.vp[0][G - 1]), as_half2(x.vp[1][G - 1])));
    need |= __hgt(__low2half(top), r_inv);
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float v = fmaxf(sc[nt][c], sc[nt][c + 2]);
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
          v = fmaxf(v, m[nt][c]);
          const float al = v == -INFINITY ? 1.f : ex2(m[nt][c] - v);
          m[nt][c] = v;
          l[nt][c] *= al;
#pragma unroll
          for (int gr = 0; gr < G; ++gr) am[nt][gr][c] *= al;
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt) o[nt][mt][c] *= al, o[nt][mt][c + 2] *= al;
        }
      float v = __low2float(top);
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, s));
      v = fminf(v, 65504.f);
      if (v > __half2float(r_inv)) {
        const float r = pow2f(-exponent_of(v) - 1), f = r / R;
        R = r;
        r_inv = __float2half_rn(1.f / r);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][mt][i] *= f;
      }
    }
    float p[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[nt][i] = ex2(sc[nt][i] - m[nt][i & 1]);
        if constexpr (kMasked) p[nt][i] = vis[nt][i] ? p[nt][i] : 0.f;  // a row that saw nothing yet has m = -inf
        l[nt][i & 1] += p[nt][i];
      }
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      const float sr[2] = {low_f16(x.vp[0][gr]) * R, low_f16(x.vp[1][gr]) * R};
      const float mv[2] = {high_f16(x.vp[0][gr]), high_f16(x.vp[1][gr])};
      uint32_t wb[NT][2], wl[NT][2];  // p s_v R as the B operand: high part, and the rest
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = p[nt][i] * sr[i >> 1];
          if constexpr (kMasked) {  // 0 * NaN stays out
            w[i] = vis[nt][i] ? w[i] : 0.f;
            am[nt][gr][i & 1] += vis[nt][i] ? p[nt][i] * mv[i >> 1] : 0.f;
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
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t sel = half ? 0x7632 : 0x5410;
        const uint32_t p01 = __byte_perm(x.v[0][gr], x.v[1][gr], sel), p23 = __byte_perm(x.v[2][gr], x.v[3][gr], sel);
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
  };

  // tiles of this warp: j, j + 4, ..; the first `whole` of the split are seen in whole by every row
  const int ntiles = k1 > k0 ? (k1 - k0 + kKv4Tile - 1) / kKv4Tile : 0;
  const int whole = k1 > k0 ? max(0, min(k1, start + r0 / grp + 1) - k0) / kKv4Tile : 0;
  int j = warp;
  advance(warp);
  if (j < whole) {
    Kv4Tile<G> x, y;
    load(x, std::false_type{}, 0);
    while (true) {  // one tile in flight while the other is worked on
      advance(kKv4Warps);
      if (j + kKv4Warps < whole) load(y, std::false_type{}, 0);
      step(x, 0, std::false_type{});
      j += kKv4Warps;
      if (j >= whole) break;
      advance(kKv4Warps);
      if (j + kKv4Warps < whole) load(x, std::false_type{}, 0);
      step(y, 0, std::false_type{});
      j += kKv4Warps;
      if (j >= whole) break;
    }
  }
  for (; j < ntiles; j += kKv4Warps) {
    Kv4Tile<G> x;
    const int p0 = k0 + j * kKv4Tile;
    load(x, std::true_type{}, k1 - p0);
    advance(kKv4Warps);
    step(x, p0, std::true_type{});
  }

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
        const float u = pow2f(20) / R;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          float* d = &sm_o[warp][n][gr * kKv4Group + g * 8 + mt * 2];
          d[0] = fmaf(o[nt][gr * 4 + mt][c], 16.f * u, am[nt][gr][c]);
          d[1] = fmaf(o[nt][gr * 4 + mt][c + 2], u, am[nt][gr][c]);
        }
      }
    }
  __syncthreads();
  for (int idx = threadIdx.x; idx < kRows * D; idx += kKv4Warps * 32) {
    const int n = idx / D, d = idx % D, r = r0 + n;
    if (r >= nrows) continue;
    float M = -INFINITY, L = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) M = fmaxf(M, sm_m[w][n]);
    const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kKv4Warps; ++w) {
      const float f = ex2(sm_m[w][n] - Mu);  // 0 for a warp that saw nothing
      L = fmaf(sm_l[w][n], f, L);
      v = fmaf(sm_o[w][n][d], f, v);
    }
    const size_t row = ((size_t)b * a.heads + kvh * grp + r % grp) * a.seq + r / grp;
    if (a.splits > 1) {
      if (d == 0) a.ml[row * a.splits + blockIdx.z] = make_float2(M, L);
      a.acc[(row * a.splits + blockIdx.z) * D + d] = v;
    } else {
      v = L == 0.f ? 0.f : v / L;
      if constexpr (OUT_BF16) static_cast<__nv_bfloat16*>(a.out)[row * D + d] = __float2bfloat16_rn(v);
      else static_cast<float*>(a.out)[row * D + d] = v;
    }
  }
}

// Merge of the splits of one query row per CTA: warp w takes splits w, w + 4, .., each lane D / 32 features;
// the four sums are added in warp order.
template <int D, bool OUT_BF16>
__global__ void __launch_bounds__(128) kv4_merge_kernel(Kv4AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = D / 32;
  __shared__ float so[4][D], sl[4];
  const long long row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = (int)(row % a.seq), b = (int)(row / a.seq / a.heads);
  const int slot = a.slots[b], start = min(a.starts[b], a.kv_len);
  // the splits that the CTA of this row had work in: up to the last row of the row's tile
  const int n = slot >= 0 && slot < a.num_slots && start >= 0 ? min(a.kv_len, start + i + 1) : 0;
  const int splits = (n + a.chunk - 1) / a.chunk;
  const float2* ml = a.ml + row * a.splits;
  float M = -INFINITY;
  for (int s = lane; s < splits; s += 32) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float Mu = M == -INFINITY ? 0.f : M;
  float L = 0.f, v[E] = {};
#pragma unroll 4
  for (int s = warp; s < splits; s += 4) {
    const float2 x = ml[s];
    const float f = ex2(x.x - Mu);
    L = fmaf(x.y, f, L);
    const float* p = a.acc + (row * a.splits + s) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = fmaf(p[e], f, v[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = v[e];
  if (lane == 0) sl[warp] = L;
  __syncthreads();
  if (threadIdx.x < D) {
    const int d = threadIdx.x;
    L = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    const float s = (so[0][d] + so[1][d]) + (so[2][d] + so[3][d]);
    const float y = L == 0.f ? 0.f : s / L;
    if constexpr (OUT_BF16) static_cast<__nv_bfloat16*>(a.out)[row * D + d] = __float2bfloat16_rn(y);
    else static_cast<float*>(a.out)[row * D + d] = y;
  }
}

// Positions per split.  Enough CTAs for four rounds of four CTAs an SM, so that uneven lengths and the
// last round cost little, and at least one tile per warp; no split where the rows fill the GPU.
static int kv4_chunk(int batch, int heads, int kv_heads, int seq, int kv_len) {
  const long rows = (long)(heads / kv_heads) * seq, per = rows <= 8 ? 8 : 16;
  const long units = (long)batch * kv_heads * ((rows + per - 1) / per);
  const long target = 4L * 4 * 148, least = kKv4Warps * kKv4Tile;
  if (kv_len <= least || units >= target / 2) return kv_len > 0 ? kv_len : 1;
  long chunk = (units * kv_len + target - 1) / target;
  chunk = (chunk + least - 1) / least * least;
  return (int)(chunk < kv_len ? chunk : kv_len);
}

template <int D, bool OB>
static int run_kv4_attention(Kv4AttnArgs a, int batch, cudaStream_t st) {
  const long rows = (long)(a.heads / a.kv_heads) * a.seq;
  const int per = rows <= 8 ? 8 : 16;
  const dim3 grid((unsigned)((rows + per - 1) / per), batch * a.kv_heads, a.splits);
  auto kern = per == 8 ? kv4_attn_kernel<D, 1, OB> : kv4_attn_kernel<D, 2, OB>;
  int rc = launch_k(kern, grid, dim3(kKv4Warps * 32), 0, st, a);
  if (rc || a.splits == 1) return rc;
  return launch_k(kv4_merge_kernel<D, OB>, dim3((unsigned)((long)batch * a.heads * a.seq)), dim3(128), 0, st, a);
}

}  // namespace ccut

using namespace ccut;

extern "C" {

size_t ccut_kv4_attention_workspace_bytes(int batch, int heads, int kv_heads, int seq, int kv_len, int head_dim) {
  if (batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || seq < 0 || kv_len < 0 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  if (batch == 0 || seq == 0 || kv_len == 0) return 256;
  const int chunk = kv4_chunk(batch, heads, kv_heads, seq, kv_len);
  const size_t sp = (kv_len + chunk - 1) / chunk;
  if (sp <= 1) return 256;
  return 256 + sp * batch * heads * seq * (head_dim + 2) * sizeof(float);
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
  if (rows > 2147483647LL || (long long)batch * kv_heads > 65535) return CCUT_ERR_UNSUPPORTED;
  const size_t need = ccut_kv4_attention_workspace_bytes(batch, heads, kv_heads, seq, kv_len, head_dim);
  if (need > 256 && (!workspace || ws_bytes < need)) return CCUT_ERR_WORKSPACE;
  if (!(scale > 0.f)) scale = 1.f / sqrtf((float)head_dim);
  const int chunk = kv4_chunk(batch, heads, kv_heads, seq, kv_len);
  Kv4AttnArgs a{q, k_codes, reinterpret_cast<const __half2*>(k_params), v_codes,
                reinterpret_cast<const __half2*>(v_params), slots, starts, heads, kv_heads, seq, max_len, kv_len,
                num_slots, slot_rows, scale, softcap, out, nullptr, nullptr, chunk,
                kv_len > 0 ? (kv_len + chunk - 1) / chunk : 1};
  if (a.splits > 1) {
    a.ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + 256);
    a.acc = reinterpret_cast<float*>(a.ml + (size_t)rows * a.splits);
  }
  const bool ob = out_dtype == CCUT_OUT_BF16;
  if (head_dim == 128)
    return ob ? run_kv4_attention<128, true>(a, batch, stream) : run_kv4_attention<128, false>(a, batch, stream);
  return ob ? run_kv4_attention<64, true>(a, batch, stream) : run_kv4_attention<64, false>(a, batch, stream);
}

}  // extern "C"
