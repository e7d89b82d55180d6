// kv4_prefill.cu -- attention of long query blocks (prompt chunks) over the 4-bit kv cache, on tcgen05.
//
// The same function as kv4_attn.cu.  Bound: tensor cores and the exponentials (4 x rows x positions x d flop
// against rows x positions exponentials: at d = 128 a tile's products and its exponentials take the same time).
//
// kv4_unpack_kernel turns the cache's rows that any query sees into fp16 once per call (value q s + m, one
// rounding to 11 bits), 2 x d x 2 bytes per position: about 3% of the products' time at 4096 rows, where
// unpacking in every CTA would repeat it per 256 rows.  A position that holds a NaN, in k or in v, gets a NaN key and
// a zero value: the key makes every row that sees it NaN, in all its features, and a masked row multiplies a zero.
// kv4_prefill_kernel: a CTA takes 256 query rows of one kv head (row r = query r / group, head r % group), two
// tiles of 128, and streams tiles of 128 positions:
// - warp 0 loads k and v tiles by TMA into a ring; warp 1 issues the MMAs (M = 128, fp32 in tensor memory):
//   S_i = Q_i K^T, then O_i += P_i V with P_i read from tensor memory, where it takes the place of S_i.
// - two warpgroups of softmax threads, one row a thread: S to registers, running maximum, exponentials, P
//   back as fp16.  While one tile's scores are worked on, the tensor cores run the other's products.
// - The maximum moves only when a score of the row passes it by 2^4, so O is rescaled a few times per row and not
//   every tile (probabilities up to 2^4 fit fp16, scaled as they are by kKv4Room); when it moves, the O of the
//   earlier tiles is complete, since S_i of a tile is issued behind P_i V of the one before.
// - With 64 features P has columns of its own: S_i of the next tile is computed while the softmax of this one
//   runs (4096 rows: 118 us, 134 in turn).  With 128 tensor memory is full, and a softmax warp waits 1400 of
//   the 3300 cycles of a step; tiles of 64 positions with two score buffers took 185 us for 158, since the
//   query operand is then read twice as often.
// Measured, 32 heads on 4 kv heads: 4096 rows from position 0, d = 128, 148 us (0.93 PFLOP/s of visible
// products), 8192 rows 494 us (1.11); d = 64 118 us.
// Roundings: q to fp16 after scaling its row's largest element to [1/2, 1) (11 bits of it, 2^-25 of the
// largest), k and v above, P to 11 bits down to 2^-25 of the maximum and 2^-36 of it absolutely, whatever the type
// of the output; scores, maximum, sums and O are fp32.
#include <math.h>

#include "kv4.cuh"
#include "tc.cuh"

namespace ccut {

constexpr int kPfRows = 128;       // query rows per tile; two tiles per CTA
constexpr int kPfTile = 128;       // positions per tile
constexpr int kPfThreads = 384;    // warps: producer, issuer, two idle, then two warpgroups of softmax
constexpr float kPfLog2e = 1.4426950408889634f;

struct PrefillArgs {
  const uint16_t* q;
  const int32_t* slots;
  const int32_t* starts;
  int heads, kv_heads, seq, kv_len, num_slots, padded;  // padded: rows per (batch row, kv head) of the unpacked cache
  float scale, softcap;
  void* out;
  int* status;
  float* part;  // [splits][rows][d + 2]: maximum, sum, output of a split
  int splits;
  long long rows;
  long long budget;  // of every wait, in cycles
};

template <int D>
struct PfSmem {
  static constexpr int kTileBytes = kPfTile * D * 2;  // q, k or v
  static constexpr int kStages = D == 128 ? 4 : 8;
  // Room in tensor memory for P beside S: S of the next tile is computed while the softmax of this one runs.
  static constexpr bool kAhead = D == 64;
  static constexpr int kBytes = 1024 + (2 + kStages) * kTileBytes;
};

struct PfBars {
  uint64_t q_raw[2], q_full[2], kv_full[8], kv_empty[8], s_full[2], s_free[2], p_half[2], p_full[2], o_full[2], drain;
  uint32_t tmem;
  int failed, loads;  // a wait ran out; k and v tiles that were sent for
};

// One thread of the (converged) warp; code behind it keeps its operands in uniform registers.
CCUT_DEVICE bool pf_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// D[tmem] (+)= A[smem] B[smem], and with A in tensor memory.
CCUT_DEVICE void pf_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
CCUT_DEVICE void pf_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// B operand stored [k][n], 64 n to a row of 128 bytes: 8-row groups of k 1024 bytes apart (stride offset), the next
// 64 n one sub-tile of 128 rows further (leading offset).
CCUT_DEVICE uint64_t pf_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFF);
  d |= (uint64_t)(kPfTile * 128 >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
CCUT_DEVICE float pf_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// To fp16, finite: a scale that was rounded up takes an appended group's top to 65536 at most, half a step above 65504.
CCUT_DEVICE __half2 pf_half2(float a, float b) {
  return __floats2half2_rn(fminf(fmaxf(a, -65504.f), 65504.f), fminf(fmaxf(b, -65504.f), 65504.f));
}

// Unpacked rows: [batch][kv_heads][padded][d] fp16 of k and of v; zeros past what the batch row sees.
template <int D>
__global__ void __launch_bounds__(256) kv4_unpack_kernel(const uint8_t* __restrict__ kc, const __half2* __restrict__ kp,
                                                         const uint8_t* __restrict__ vc, const __half2* __restrict__ vp,
                                                         const int32_t* __restrict__ slots,
                                                         const int32_t* __restrict__ starts, int kv_heads, int seq,
                                                         int kv_len, int max_len, long long slot_rows, int num_slots,
                                                         int padded, uint4* __restrict__ k16, uint4* __restrict__ v16,
                                                         int* status) {
  pdl_wait();
  pdl_trigger();
  constexpr int W = D / 8, G = D / kKv4Group;
  const int b = blockIdx.z, h = blockIdx.y;
  if (blockIdx.x == 0 && b == 0 && h == 0 && threadIdx.x == 0) *status = 0;
  const int slot = slots[b], start = starts[b];
  const int seen = slot >= 0 && slot < num_slots && start >= 0 ? min(kv_len, min(start, kv_len) + seq) : 0;
  const int idx = blockIdx.x * 256 + threadIdx.x, pos = idx / W, w = idx % W;
  if (pos >= padded || pos >= (seen + kPfTile - 1) / kPfTile * kPfTile) return;  // tiles past the last are not read
  uint32_t k[4] = {0, 0, 0, 0}, v[4] = {0, 0, 0, 0};
  if (pos < seen) {
    const size_t row = (size_t)slot * (size_t)slot_rows + (size_t)h * max_len + pos;
    bool bad = false;
    float2 pk{}, pv{};
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float2 a = __half22float2(kp[row * G + g]), c = __half22float2(vp[row * G + g]);
      bad |= !(fabsf(a.x) + fabsf(a.y) + fabsf(c.x) + fabsf(c.y) < INFINITY);
      if (g == w / 8) pk = a, pv = c;
    }
    const uint32_t wk = reinterpret_cast<const uint32_t*>(kc)[row * W + w], wv = reinterpret_cast<const uint32_t*>(vc)[row * W + w];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 hk = pf_half2(kv4_value((wk >> (8 * i)) & 15, pk.x, pk.y), kv4_value((wk >> (8 * i + 4)) & 15, pk.x, pk.y));
      const __half2 hv = pf_half2(kv4_value((wv >> (8 * i)) & 15, pv.x, pv.y), kv4_value((wv >> (8 * i + 4)) & 15, pv.x, pv.y));
      k[i] = bad ? 0x7FFF7FFFu : *reinterpret_cast<const uint32_t*>(&hk);
      v[i] = bad ? 0u : *reinterpret_cast<const uint32_t*>(&hv);
    }
  }
  const size_t at = (((size_t)b * kv_heads + h) * padded + pos) * W + w;
  k16[at] = make_uint4(k[0], k[1], k[2], k[3]);
  v16[at] = make_uint4(v[0], v[1], v[2], v[3]);
}

template <int D, bool OUT_BF16>
__global__ void __launch_bounds__(kPfThreads, 1)
    kv4_prefill_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                       const __grid_constant__ PrefillArgs a) {
  using SM = PfSmem<D>;
  constexpr int kChunks = D / 64;  // sub-tiles of 64 features, 128 rows of 128 bytes each
  constexpr int kSub = kPfTile * 128;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  __shared__ PfBars bars;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.q_raw[i], kPfRows);
      mbar_init(&bars.q_full[i], kPfRows);
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.s_free[i], kPfRows);
      mbar_init(&bars.p_half[i], kPfRows);
      mbar_init(&bars.p_full[i], kPfRows);
      mbar_init(&bars.o_full[i], 1);
    }
    for (int i = 0; i < SM::kStages; ++i) {
      mbar_init(&bars.kv_full[i], 1);
      mbar_init(&bars.kv_empty[i], 1);
    }
    mbar_init(&bars.drain, 1);
    bars.failed = bars.loads = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tc::tmem_alloc(&bars.tmem, 512);
    tc::tmem_relinquish();
  }
  const int grp = a.heads / a.kv_heads, nrows = grp * a.seq;
  const int b = blockIdx.y / a.kv_heads, kvh = blockIdx.y % a.kv_heads;
  const int r0 = (gridDim.x - 1 - blockIdx.x) * 2 * kPfRows;  // the longest first
  const int tr = threadIdx.x & 127, my_tile = warp >= 8, my_r = r0 + my_tile * kPfRows + tr;  // a softmax thread's query row
  const bool live = warp >= 4 && my_r < nrows;
  const int my_s = my_r / grp;
  const int row = (b * a.heads + kvh * grp + my_r % grp) * a.seq + my_s;  // of q and out; rows fit 31 bits
  uint8_t* q_s = smem;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  pdl_wait();
  pdl_trigger();
  // A tile's rows of q come by one bulk copy per head, whose rows are neighbours (16-byte loads, each lane in its own
  // row, took 2000 cycles a CTA more); the heads follow one another from the first row's.
  const int have = min(kPfRows, nrows - (r0 + my_tile * kPfRows)), each = have / grp, more = have % grp;
  if (warp >= 4) {
    if (tr < min(grp, have)) {  // my_r is the first row of its head
      const int bytes = ((have - 1 - tr) / grp + 1) * D * 2;
      mbar_arrive_expect_tx(&bars.q_raw[my_tile], bytes);
      bulk_g2s(q_s + my_tile * SM::kTileBytes + (tr * each + min(tr, more)) * (D * 2), a.q + (size_t)row * D, bytes,
               &bars.q_raw[my_tile]);
    } else {
      mbar_arrive(&bars.q_raw[my_tile]);
    }
  }
  const int slot = a.slots[b], start0 = a.starts[b];
  const bool valid = slot >= 0 && slot < a.num_slots && start0 >= 0;
  const int start = min(start0, a.kv_len);
  const int last_row = min(nrows, r0 + 2 * kPfRows) - 1;
  const int seen = valid ? min(a.kv_len, start + last_row / grp + 1) : 0;  // by any row of this CTA
  const int all = (seen + kPfTile - 1) / kPfTile;
  const int tile0 = (int)((long long)all * blockIdx.z / a.splits), tile1 = (int)((long long)all * (blockIdx.z + 1) / a.splits);
  const int n = tile1 - tile0;
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars.tmem, 0);
  volatile int* failed = &bars.failed;
  // columns: S_0, S_1, O_0, O_1, P_0, P_1 (P_i in the first half of S_i where there is no room)
  auto s_col = [&](int i) { return tmem + i * kPfTile; };
  auto o_col = [&](int i) { return tmem + 2 * kPfTile + i * D; };
  auto p_col = [&](int i) { return SM::kAhead ? tmem + 2 * kPfTile + 2 * D + i * (kPfTile / 2) : s_col(i); };
  uint8_t* ring = smem + 2 * SM::kTileBytes;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    const bool ok = mbar_wait(bar, parity, a.status, a.budget);
    if (!ok) *failed = 1;
    return ok && !*failed;
  };

  // 256 x 208 + 128 x 88 registers of the 384 x 168 of the launch; one instruction per warpgroup
  if (warp < 4) {
  tc::setmaxnreg_dec<88>();
  if (warp == 0) {
    if (lane == 0 && n > 0) {
      asm volatile("fence.proxy.async;" ::: "memory");  // the unpacked cache was written through the generic proxy
      tc::prefetch_tmap(&kmap);
      tc::prefetch_tmap(&vmap);
      const int row = (int)(((long long)b * a.kv_heads + kvh) * a.padded) + tile0 * kPfTile;
      int st = 0, ph = 1, loads = 0;  // the ring's next stage; its first use finds it empty
      auto load = [&](const CUtensorMap* map, int j) {
        if (!wait(&bars.kv_empty[st], ph)) return false;
        mbar_arrive_expect_tx(&bars.kv_full[st], SM::kTileBytes);
        for (int c = 0; c < kChunks; ++c)
          tc::tma_load_2d(ring + st * SM::kTileBytes + c * kSub, map, c * 64, row + j * kPfTile, &bars.kv_full[st]);
        ++loads;
        if (++st == SM::kStages) st = 0, ph ^= 1;
        return true;
      };
      bool ok = !SM::kAhead || load(&kmap, 0);  // k j + 1 before v j where S runs ahead, else k j
      for (int j = 0; ok && j < n; ++j) {
        const int k = SM::kAhead ? j + 1 : j;
        ok = (k >= n || load(&kmap, k)) && load(&vmap, j);
      }
      bars.loads = loads;
    }
  } else if (warp == 1 && n > 0) {
    // The whole warp walks through the steps and one lane issues: a divergent lane could not use the uniform
    // registers that the MMAs take their operands from, and moving them there took longer than the MMAs.
    const uint32_t idesc_s = tc::idesc_f16_m128(kPfTile);
    const uint32_t idesc_o = tc::idesc_f16_m128(D) | (1u << 16);  // B is [k][n]
    auto spin = [&](uint64_t* bar, uint32_t parity) {  // its wake-up is on the critical path
      const bool ok = mbar_spin(bar, parity, a.status, a.budget);
      if (!ok) *failed = 1;
      return __all_sync(0xffffffffu, ok && !*failed) != 0;
    };
    const uint64_t q_desc = tc::sdesc_sw128(smem_u32(q_s));
    const uint64_t k_desc = tc::sdesc_sw128(smem_u32(ring)), v_desc = pf_desc_mn(smem_u32(ring));
    auto scores = [&](int i, int st, bool free_k) {  // S_i = Q_i K^T, K in the ring's stage st
      const uint64_t q0 = q_desc + (uint64_t)(i * (SM::kTileBytes >> 4)), k0 = k_desc + (uint64_t)(st * (SM::kTileBytes >> 4));
      if (pf_elect()) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t off = (ks >> 2) * (kSub >> 4) + (ks & 3) * (32 >> 4);
          pf_mma_ss(s_col(i), q0 + off, k0 + off, idesc_s, ks > 0);
        }
        tc::commit(&bars.s_full[i]);
        if (free_k) tc::commit(&bars.kv_empty[st]);
      }
      __syncwarp();
    };
    auto products = [&](int i, int k0, int k1, int sv, bool first) {  // O_i (+)= P_i V over k16 steps k0 ..
      const uint64_t v0 = v_desc + (uint64_t)(sv * (SM::kTileBytes >> 4));
      if (pf_elect()) {
#pragma unroll
        for (int ks = k0; ks < k1; ++ks)
          pf_mma_ts(o_col(i), p_col(i) + ks * 8, v0 + ks * (2048 >> 4), idesc_o, ks > 0 || !first);
      }
    };
    auto advance = [](int& st, int& ph) {
      if (++st == SM::kStages) st = 0, ph ^= 1;
    };
    bool ok = spin(&bars.q_full[0], 0) && spin(&bars.kv_full[0], 0);
    tc::fence_after_sync();
    if (ok) scores(0, 0, false);
    ok = ok && spin(&bars.q_full[1], 0);
    tc::fence_after_sync();
    if (ok) scores(1, 0, true);
    int st = 1, ph = 0;  // the ring's next stage and the parity of its use
    if constexpr (SM::kAhead) {
      // S_0 of tile j + 1, P_1 V of j - 1, S_1 of j + 1, P_0 V of j: what two tiles half a step apart ask for in turn
      auto join = [&](int i, int j, int sv) {
        if (!spin(&bars.p_full[i], j & 1)) return false;
        tc::fence_after_sync();
        products(i, 0, kPfTile / 16, sv, j == 0);
        if (pf_elect()) {
          if (i == 1) tc::commit(&bars.kv_empty[sv]);
          tc::commit(&bars.o_full[i]);
        }
        __syncwarp();
        return true;
      };
      int sv = 0;  // of v tile j - 1
      for (int j = 0; ok && j < n; ++j) {
        int sk = 0;
        if (j + 1 < n) {
          sk = st;
          if (!(ok = spin(&bars.kv_full[sk], ph) && spin(&bars.s_free[0], j & 1))) break;
          advance(st, ph);
          tc::fence_after_sync();
          scores(0, sk, false);
        }
        if (j > 0 && !(ok = join(1, j - 1, sv))) break;
        if (j + 1 < n) {
          if (!(ok = spin(&bars.s_free[1], j & 1))) break;
          tc::fence_after_sync();
          scores(1, sk, true);
        }
        sv = st;
        if (!(ok = spin(&bars.kv_full[sv], ph))) break;
        advance(st, ph);
        if (!(ok = join(0, j, sv))) break;
      }
      if (ok) join(1, n - 1, sv);
    } else {
      for (int j = 0; ok && j < n; ++j) {
        const int sv = st;
        if (!(ok = spin(&bars.kv_full[sv], ph))) break;
        advance(st, ph);
        const int sk = st;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (!(ok = spin(&bars.p_half[i], j & 1))) break;
          tc::fence_after_sync();
          products(i, 0, kPfTile / 32, sv, j == 0);
          __syncwarp();
          if (!(ok = spin(&bars.p_full[i], j & 1))) break;
          tc::fence_after_sync();
          products(i, kPfTile / 32, kPfTile / 16, sv, false);
          if (pf_elect()) {
            if (i == 1) tc::commit(&bars.kv_empty[sv]);
            if (j + 1 == n) tc::commit(&bars.o_full[i]);
          }
          __syncwarp();
          if (j + 1 < n) {
            if (i == 0 && !(ok = spin(&bars.kv_full[sk], ph))) break;
            tc::fence_after_sync();
            scores(i, sk, i == 1);
          }
        }
        if (j + 1 < n) advance(st, ph);
      }
    }
  }
  } else {
    tc::setmaxnreg_inc<208>();
    const int i = (warp - 4) >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = s_col(i) + lanes, p_addr = p_col(i) + lanes, o_addr = o_col(i) + lanes;
    const int lim = live ? start + my_s : a.kv_len;  // last visible position
    // The thread takes its row of q and writes it back as fp16, scaled by a power of two, into the swizzled tile, its
    // 16-byte pieces in an order c ^ turn in which eight threads meet every bank once both in the plain rows and in
    // the swizzled ones: turn is a linear map of tr & 7 over GF(2) (times x in GF(8)) for which turn and turn ^ tr
    // are both one to one.
    float fr = 0.f;
    bool ok = wait(&bars.q_raw[i], 0);  // also where there is nothing to see: the copy must have landed
    ok = !__any_sync(0xffffffffu, !ok);
    if (n > 0) {
      uint8_t* const tile = q_s + i * SM::kTileBytes;
      const uint8_t* const mine = tile + (tr % grp * each + min(tr % grp, more) + tr / grp) * (D * 2);
      const int turn = ((tr << 1) & 7) ^ (tr & 4 ? 3 : 0);
      uint4 u[D / 8];
      float mx = 0.f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        u[c] = live ? *reinterpret_cast<const uint4*>(mine + ((c ^ turn) << 4)) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mx = fmaxf(mx, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xFFFF0000u))));
      }
      const int ex = min(max((int)((__float_as_uint(mx) >> 23) & 255) - 126, -90), 90);  // |q| 2^-ex in [1/2, 1)
      const float f = __int_as_float((127 - ex) << 23);
      fr = __int_as_float((127 + ex) << 23) * (a.scale * kPfLog2e);
      asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");  // the tile's rows are all in registers
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __half2 h = __floats2half2_rn(__uint_as_float(w[e] << 16) * f, __uint_as_float(w[e] & 0xFFFF0000u) * f);
          o[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        const int k = c ^ turn;
        *reinterpret_cast<uint4*>(tile + (k >> 3) * kSub + tr * 128 + (((k ^ tr) & 7) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      tc::fence_proxy_async_smem();
      mbar_arrive(&bars.q_full[i]);
    }
    float m = -INFINITY, l = 0.f;  // the maximum less kKv4Room: l and O are 2^kKv4Room larger, and so are P's
    for (int j = 0; ok && j < n; ++j) {
      ok = wait(&bars.s_full[i], j & 1);
      ok = !__any_sync(0xffffffffu, !ok);
      if (!ok) break;
      tc::fence_after_sync();
      uint32_t x[4][32];
      __syncwarp();
#pragma unroll
      for (int c = 0; c < 4; ++c) tc::ld_32x32b_x32(s_addr + c * 32, x[c]);
      tc::wait_ld();
      if constexpr (SM::kAhead) {
        tc::fence_before_sync();
        mbar_arrive(&bars.s_free[i]);
      }
      const int p0 = (tile0 + j) * kPfTile;
      float f = fr;
      if (a.softcap > 0.f) {
        f = 1.f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            x[c][e] = __float_as_uint(tanhf(__uint_as_float(x[c][e]) * (fr / kPfLog2e) / a.softcap) * (a.softcap * kPfLog2e));
      }
      if (__any_sync(0xffffffffu, p0 + kPfTile - 1 > min(lim, seen - 1))) {
        const int vis = min(lim, seen - 1) - p0;  // columns up to this one
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c * 32 + e > vis) x[c][e] = 0xFF800000u;
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; e += 2)
#pragma unroll
        for (int c = 0; c < 4; ++c) top[c] = pf_max3(top[c], __uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1]));
      const float mt = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * f;
      if constexpr (SM::kAhead) {  // P and O are free: the product of the tile before is done
        if (j > 0) {
          ok = wait(&bars.o_full[i], (j - 1) & 1);
          ok = !__any_sync(0xffffffffu, !ok);
          tc::fence_after_sync();
        }
      }
      if (__any_sync(0xffffffffu, mt > m + (kKv4Room + kKv4Lag))) {
        const float mn = mt > m + (kKv4Room + kKv4Lag) ? mt - kKv4Room : m, al = mn == m ? 1.f : pf_ex2(m - mn);  // by the row's own scores
        m = mn;
        l *= al;
        __syncwarp();
        if (j > 0) {  // O of the tiles before is complete (else than above: S_i was issued behind its last product)
#pragma unroll
          for (int c = 0; c < D; c += 16) {
            uint32_t y[16];
            tc::ld_32x32b_x16(o_addr + c, y);
            tc::wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * al);
            tc::st_32x32b_x16(o_addr + c, y);
          }
        }
      }
      const float mu = m == -INFINITY ? 0.f : m;
      __syncwarp();
      const u64 f2 = pf_pair(f, f), mu2 = pf_pair(-mu, -mu);
      u64 sum[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        uint32_t p[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const uint32_t* xe = &x[c + (e >> 4)][(e & 15) * 2];
          const u64 t = pf_fma2(pf_pair(__uint_as_float(xe[0]), __uint_as_float(xe[1])), f2, mu2);
          float y0, y1;
          pf_unpair(t, y0, y1);
          y0 = pf_ex2(y0), y1 = pf_ex2(y1);
          sum[e & 1] = pf_add2(sum[e & 1], pf_pair(y0, y1));
          const __half2 h = __floats2half2_rn(y0, y1);
          p[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        tc::st_32x32b_x32(p_addr + c * 16, p);
        tc::wait_st();
        tc::fence_before_sync();
        if (c > 0) mbar_arrive(&bars.p_full[i]);
        else if (!SM::kAhead) mbar_arrive(&bars.p_half[i]);  // the product of the first half can begin
      }
      float l0, l1;
      pf_unpair(pf_add2(sum[0], sum[1]), l0, l1);
      l += l0 + l1;
    }
    if (n > 0 && ok) ok = wait(&bars.o_full[i], SM::kAhead ? (n - 1) & 1 : 0);
    ok = !__any_sync(0xffffffffu, !ok);
    tc::fence_after_sync();
    const float inv = l == 0.f ? 0.f : 1.f / l;
    // a row of bf16 outputs, rows 16 bytes more than their size apart: tile 0's in the place of the query tiles (every S
    // was issued before its last product), tile 1's behind them, where nothing is left to be read.  Tile 0's last rows pass
    // the end of its query tile: it is the products that order them behind the copy of tile 1's, so rows that come
    // without products (zeros) go straight to memory.
    const bool staged = n > 0 && ok;
    uint8_t* const mine = q_s + (i * kPfRows + tr) * (D * 2 + 16);
#pragma unroll
    for (int c = 0; c < D; c += 32) {
      uint32_t y[32];
      __syncwarp();
      if (staged) {
        tc::ld_32x32b_x32(o_addr + c, y);
        tc::wait_ld();
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) y[e] = 0;
      }
      if (!live) {
        // a row past the last is not written
      } else if (a.splits > 1) {
        float* p = a.part + ((size_t)blockIdx.z * a.rows + row) * (D + 4);
        if (c == 0) p[0] = m, p[1] = l;
#pragma unroll
        for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(p + 4 + c + e) = make_uint4(y[e], y[e + 1], y[e + 2], y[e + 3]);
      } else if constexpr (OUT_BF16) {  // by a bulk copy of the row from shared memory, as above
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint32_t o[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(y[e + 2 * q]) * inv, __uint_as_float(y[e + 2 * q + 1]) * inv);
            o[q] = *reinterpret_cast<const uint32_t*>(&h);
          }
          if (staged) *reinterpret_cast<uint4*>(mine + (c + e) * 2) = make_uint4(o[0], o[1], o[2], o[3]);
          else *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (size_t)row * D + c + e) = make_uint4(0, 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<float4*>(static_cast<float*>(a.out) + (size_t)row * D + c + e) =
              make_float4(__uint_as_float(y[e]) * inv, __uint_as_float(y[e + 1]) * inv, __uint_as_float(y[e + 2]) * inv,
                          __uint_as_float(y[e + 3]) * inv);
      }
    }
    if constexpr (OUT_BF16) {
      if (live && a.splits == 1 && staged) {
        tc::fence_proxy_async_smem();
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;\n\t"
                     "cp.async.bulk.wait_group.read 0;" ::"l"(static_cast<uint16_t*>(a.out) + (size_t)row * D),
                     "r"(smem_u32(mine)), "r"(D * 2)
                     : "memory");
      }
    }
    tc::fence_before_sync();
  }
  __syncthreads();
  if (*failed) {  // copies and products that nobody waited for end before shared and tensor memory go, or a second passes
    if (threadIdx.x == 0) {
      for (int i = 0; i < 2; ++i) mbar_wait(&bars.q_raw[i], 0, a.status);
      for (int u = max(0, bars.loads - SM::kStages); u < bars.loads; ++u)
        mbar_wait(&bars.kv_full[u % SM::kStages], u / SM::kStages & 1, a.status);
    }
    if (warp == 1) {
      if (pf_elect()) tc::commit(&bars.drain);
      __syncwarp();
      mbar_wait(&bars.drain, 0, a.status);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins the splits of a row, one warp each, in split order.
template <int D, bool OUT_BF16>
__global__ void __launch_bounds__(256) kv4_prefill_merge_kernel(PrefillArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int E = D / 32;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  float M = -INFINITY, L = 0.f, v[E] = {};
  for (int s = 0; s < a.splits; ++s) {
    const float* p = a.part + ((size_t)s * a.rows + row) * (D + 4);
    const float m = p[0], top = fmaxf(M, m), base = top == -INFINITY ? 0.f : top;
    const float f = pf_ex2(M - base), g = pf_ex2(m - base);
    M = top;
    L = fmaf(L, f, p[1] * g);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = fmaf(v[e], f, p[4 + lane + 32 * e] * g);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if constexpr (OUT_BF16) static_cast<__nv_bfloat16*>(a.out)[row * D + lane + 32 * e] = __float2bfloat16_rn(v[e] * inv);
    else static_cast<float*>(a.out)[row * D + lane + 32 * e] = v[e] * inv;
  }
}

static long long pf_padded(int kv_len) { return ((long long)kv_len + kPfTile - 1) / kPfTile * kPfTile; }
static long long pf_row_tiles(int heads, int kv_heads, int seq) {
  return ((long long)(heads / kv_heads) * seq + 2 * kPfRows - 1) / (2 * kPfRows);
}
// Splits of the positions: one CTA an SM, at least four tiles each.
static int pf_splits(int batch, int heads, int kv_heads, int seq, int kv_len) {
  const long long units = pf_row_tiles(heads, kv_heads, seq) * kv_heads * batch, tiles = pf_padded(kv_len) / kPfTile;
  long long sp = units > 0 ? 148 / units : 1;
  if (sp > tiles / 4) sp = tiles / 4;
  return sp < 1 ? 1 : sp > 16 ? 16 : (int)sp;
}

bool kv4_prefill_fits(int batch, int heads, int kv_heads, int seq, int kv_len) {
  const long long rows = (long long)(heads / kv_heads) * seq;
  return rows >= kKv4LongRows && kv_len > 0 && (double)batch * kv_heads * pf_padded(kv_len) < 2147483647.0 &&
         (long long)batch * kv_heads <= 65535 && batch <= 65535 && kv_heads <= 65535 &&
         pf_padded(kv_len) <= 2147483647LL / 16;
}
size_t kv4_prefill_workspace(int batch, int heads, int kv_heads, int seq, int kv_len, int head_dim) {
  const int sp = pf_splits(batch, heads, kv_heads, seq, kv_len);
  const size_t cache = (size_t)batch * kv_heads * pf_padded(kv_len) * head_dim * 2 * 2;
  return 256 + cache + (sp > 1 ? (size_t)sp * batch * heads * seq * (head_dim + 4) * sizeof(float) : 0);
}

static thread_local long long g_pf_budget = kWaitBudgetCycles;
long long kv4_wait_budget(long long cycles) {
  const long long was = g_pf_budget;
  g_pf_budget = cycles;
  return was;
}

template <int D, bool OB>
static int run_prefill(const Kv4Cache& c, PrefillArgs a, int batch, void* workspace, int* status, cudaStream_t st) {
  const size_t rows = (size_t)batch * a.kv_heads * a.padded;
  uint8_t* k16 = static_cast<uint8_t*>(workspace) + 256;
  uint8_t* v16 = k16 + rows * D * 2;
  int* const word = static_cast<int*>(workspace);
  a.status = status ? status : word;
  a.part = reinterpret_cast<float*>(v16 + rows * D * 2);
  CUtensorMap kmap, vmap;
  int rc = encode_rows_map(&kmap, k16, (int)rows, D, kPfTile);
  if (!rc) rc = encode_rows_map(&vmap, v16, (int)rows, D, kPfTile);
  if (rc) return rc;
  rc = launch_k(kv4_unpack_kernel<D>, dim3((unsigned)(((long long)a.padded * (D / 8) + 255) / 256), a.kv_heads, batch),
                dim3(256), 0, st, c.kc, c.kp, c.vc, c.vp, a.slots, a.starts, a.kv_heads, a.seq, a.kv_len, c.max_len,
                c.slot_rows, a.num_slots, a.padded, reinterpret_cast<uint4*>(k16), reinterpret_cast<uint4*>(v16), word);
  if (rc) return rc;
  static std::atomic<uint64_t> smem_set{0};  // devices with the limit raised
  rc = ensure_smem_limit(kv4_prefill_kernel<D, OB>, PfSmem<D>::kBytes, smem_set);
  if (rc) return rc;
  const dim3 grid((unsigned)pf_row_tiles(a.heads, a.kv_heads, a.seq), batch * a.kv_heads, a.splits);
  rc = launch_k(kv4_prefill_kernel<D, OB>, grid, dim3(kPfThreads), PfSmem<D>::kBytes, st, kmap, vmap, a);
  if (rc || a.splits == 1) return rc;
  return launch_k(kv4_prefill_merge_kernel<D, OB>, dim3((unsigned)((a.rows + 7) / 8)), dim3(256), 0, st, a);
}

int launch_kv4_prefill(const Kv4Cache& c, const uint16_t* q, const int32_t* slots, const int32_t* starts, int batch,
                       int heads, int kv_heads, int seq, int head_dim, int kv_len, int num_slots, float scale,
                       float softcap, void* out, bool out_bf16, void* workspace, int* status, cudaStream_t st) {
  PrefillArgs a{q, slots, starts, heads, kv_heads, seq, kv_len, num_slots, (int)pf_padded(kv_len), scale, softcap, out,
                nullptr, nullptr, pf_splits(batch, heads, kv_heads, seq, kv_len), (long long)batch * heads * seq,
                g_pf_budget};
  if (head_dim == 128)
    return out_bf16 ? run_prefill<128, true>(c, a, batch, workspace, status, st)
                    : run_prefill<128, false>(c, a, batch, workspace, status, st);
  return out_bf16 ? run_prefill<64, true>(c, a, batch, workspace, status, st)
                  : run_prefill<64, false>(c, a, batch, workspace, status, st);
}

}  // namespace ccut
