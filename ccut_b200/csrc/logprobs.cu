// logprobs.cu -- log probability, entropy and rank of given tokens, and the top alternatives.
//
// Per row x of vocab logits and its token t (natural logarithms, fp32 sums):
//   m = max x,  S = sum_v e^(x_v - m),  W = sum_v e^(x_v - m) (x_v - m),
//   logprob = x_t - m - log S,  entropy = log S - W / S,
//   rank = 1 + #{v: x_v > x_t} + #{v < t: x_v = x_t},
//   top n by (value descending, index ascending) with their log probabilities.
//
// Bound: HBM, each logit read once.  A warp streams a contiguous part of a row in rounds of 512 logits
// (16 a lane, the next round's loads in flight): about eight instructions a logit, so that the reading
// stays in front.
// - m moves once a round of a lane: the 16 logits' maximum first, then one exponential each; S and W are
//   packed pairs (fma.rn.f32x2).  A lane that finds a new maximum rescales S and W, W by
//   e^d (W + S d), d = m_old - m_new.
// - rank: x >= x_t counts before t, x >= the next float above x_t behind it; only the round that holds t
//   compares indices.
// - Top n: each warp keeps its 32 best as 64-bit keys (order of the value, then of the index) sorted
//   over its lanes.  One vote a round asks whether any lane's maximum reaches the n-th best; if so the
//   logits that do are inserted one by one, each by a vote for its place and one shift of the lanes.
//   The first list is the first round's 32 lane maxima.
//   Warps of one row publish their ceil(n / warps)-th best; the least of these is a bar for all.
// Few rows take 8 warps in each of up to 16 CTAs, a cluster, joined through its shared memory (one launch; with
// 37 CTAs a row and a second kernel that joined them, 8 rows of 151936 took 13.3 us, here 11.7, 7.2 without alternatives); many rows take fewer
// warps each, since every warp has to find its own best from the start.
#include <math.h>

#include "host.cuh"
#include "tc.cuh"

namespace ccut {

constexpr int kLpWarps = 8;
constexpr int kLpRound = 512;    // logits a warp takes in a round
constexpr int kLpCluster = 16;   // CTAs per row at most
constexpr float kL2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
typedef unsigned long long u64;

struct LpArgs {
  const void* x;
  int vocab;
  long long ld, rows;
  const int32_t* tokens;
  int top_n, wpr, ctas;  // warps per row in a CTA; CTAs per row, a cluster (then all warps of a CTA are its row's)
  float *logprob, *entropy;
  int32_t *rank, *top_ids;
  float* top_lp;
};

// The order of logits as integers: descending value is descending key, -0 equals +0, NaN comes last.
CCUT_DEVICE int order_key(float x) {
  if (isnan(x)) return -0x7FFFFFFF - 1;
  const int b = __float_as_int(x + 0.f);
  return b < 0 ? b ^ 0x7FFFFFFF : b;
}
CCUT_DEVICE u64 entry_of(float x, int i) {  // 0 is no entry
  return ((u64)((uint32_t)order_key(x) ^ 0x80000000u) << 32) | (0xFFFFFFFFu - (uint32_t)i);
}
CCUT_DEVICE float entry_value(u64 e) {
  const int k = (int)((uint32_t)(e >> 32) ^ 0x80000000u);
  return k == -0x7FFFFFFF - 1 ? __int_as_float(0x7FFFFFFF) : __int_as_float(k < 0 ? k ^ 0x7FFFFFFF : k);
}
CCUT_DEVICE int entry_index(u64 e) { return (int)(0xFFFFFFFFu - (uint32_t)e); }

// Sorted over the lanes, descending: exchanges at distance j of the bitonic network; `up`: this lane's pair ascends.
template <class T>
CCUT_DEVICE T exchange(T v, int j, bool up, int lane) {
  const T o = __shfl_xor_sync(0xffffffffu, v, j);
  const bool low = (lane & j) == 0;          // the lane that keeps the larger when descending
  return (low != up) == (v > o) ? v : o;
}
template <class T>
CCUT_DEVICE T sort32(T v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) v = exchange(v, j, k < 32 && (lane & k) != 0, lane);
  return v;
}
// The 32 largest of two descending lists, descending.
CCUT_DEVICE u64 merge32(u64 a, u64 b, int lane) {
  const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
  u64 v = a > r ? a : r;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) v = exchange(v, j, false, lane);
  return v;
}

CCUT_DEVICE float lp_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CCUT_DEVICE u64 pair(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
CCUT_DEVICE void unpair(u64 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
CCUT_DEVICE u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
CCUT_DEVICE u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
CCUT_DEVICE u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
CCUT_DEVICE float max_nan(float a, float b) {  // NaN when either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

CCUT_DEVICE float at_least(float a, float b) {  // 1 or 0
  float r;
  asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <bool BF16>
CCUT_DEVICE float logit(const void* x, long long i) {
  if constexpr (BF16) return __uint_as_float((uint32_t) static_cast<const uint16_t*>(x)[i] << 16);
  else return static_cast<const float*>(x)[i];
}

// Maximum, S and W (log2 units) of a set of logits.
struct LpSum {
  float m = -INFINITY, s = 0.f, w = 0.f;
  CCUT_DEVICE void move(float to) {  // to >= m
    const float d = m == -INFINITY ? 0.f : (m - to) * kL2e, f = m == -INFINITY ? 0.f : lp_ex2(d);
    w = f * fmaf(s, fmaxf(d, -1000.f), w);  // f is 0 long before the bound
    s *= f;
    m = to;
  }
  CCUT_DEVICE void join(LpSum o) {
    if (o.m > m) move(o.m);
    else if (m > o.m) o.move(m);
    s += o.s;
    w += o.w;
  }
};

// The answers of a row from its joined state (one warp).
template <bool BF16, bool TOP>
CCUT_DEVICE void lp_finish(const LpArgs& a, long long row, const LpSum& sum, int count, u64 list, int lane) {
  const float log_s = logf(sum.s);
  if (lane == 0) {
    const int t = a.tokens[row];
    const bool has = t >= 0 && t < a.vocab;
    const char* base = static_cast<const char*>(a.x) + row * a.ld * (BF16 ? 2 : 4);
    a.logprob[row] = has ? (logit<BF16>(base, t) - sum.m) - log_s : __int_as_float(0x7FFFFFFF);
    a.entropy[row] = log_s - sum.w * kLn2 / sum.s;
    a.rank[row] = has ? count + 1 : 0;
  }
  if constexpr (TOP) {
    if (lane < a.top_n) {
      a.top_ids[row * a.top_n + lane] = entry_index(list);
      a.top_lp[row * a.top_n + lane] = (entry_value(list) - sum.m) - log_s;
    }
  }
}

// Joins the states of each `n` (a power of two) consecutive warps into the first of them, pairwise.  Whole CTA.
template <bool TOP, class Stats, class Lists>
CCUT_DEVICE void lp_tree(LpSum& sum, int& count, u64& list, Stats& stats, Lists& lists, int warp, int lane, int n) {
  for (int s = 1; s < n; s <<= 1) {
    if (warp % (2 * s) == s) {
      if (lane == 0) stats[warp] = make_float4(sum.m, sum.s, sum.w, __int_as_float(count));
      if constexpr (TOP) lists[warp][lane] = list;
    }
    __syncthreads();
    if (warp % (2 * s) == 0) {
      const float4 y = stats[warp + s];
      LpSum o;
      o.m = y.x, o.s = y.y, o.w = y.z;
      sum.join(o);
      count += __float_as_int(y.w);
      if constexpr (TOP) list = merge32(list, lists[warp + s][lane], lane);
    }
  }
}

template <bool TOP>
struct LpWarp {  // a warp's state
  LpSum sum;
  int count = 0;  // of the rank, per lane
  u64 list = 0, bar = 0;
  float bar_value = -INFINITY;  // logits below it are not among the best
  bool first = true;
  volatile float *row_bar, *mine;  // shared memory: the row's warps' published values, this warp's
  int share;                       // ceil(top_n / warps of the row in this CTA)

  CCUT_DEVICE void insert(u64 e, int lane) {  // e the same in every lane
    const int at = __popc(__ballot_sync(0xffffffffu, list > e));
    const u64 before = __shfl_up_sync(0xffffffffu, list, 1);
    list = lane < at ? list : lane == at ? e : before;
  }
  CCUT_DEVICE void raise(int top_n, int lane) {
    const u64 nth = __shfl_sync(0xffffffffu, list, top_n - 1);
    if (nth > bar) {
      bar = nth;
      bar_value = entry_value(nth);
    }
    if (lane == share - 1 && list) {
      const float v = entry_value(list);
      mine[0] = isnan(v) ? -INFINITY : v;  // NaN comes last in the order: it bars nothing, nor does its warp
    }
  }
  // At least `share` logits of each of the row's `wpr` warps here reach its published value: at least top_n reach
  // the least of them.
  CCUT_DEVICE void look(int wpr) {
    float least = row_bar[0];
    for (int w = 1; w < wpr; ++w) least = fminf(least, row_bar[w]);
    if (least > bar_value) {
      bar_value = least;
      bar = entry_of(least, -1) & ~0xFFFFFFFFull;  // every logit of this value passes
    }
  }

  // One round: 16 logits a lane; index(i) of logit i; kChecked: those with !valid(i) do not exist.
  template <bool kChecked, class Index, class Valid>
  CCUT_DEVICE void round(const float (&x)[16], Index index, Valid valid, int begin, int end, int t, float xt, float above,
                         int top_n, int lane) {
    float top = -INFINITY, low = INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!kChecked || valid(i)) top = fmaxf(top, x[i]), low = fminf(low, x[i]);
    if (top > sum.m) sum.move(top);
    const float mu = sum.m == -INFINITY ? 0.f : sum.m;
    const u64 neg = pair(-mu, -mu), scale = pair(kL2e, kL2e);
    u64 s2 = 0, w2 = 0;
    auto terms = [&](auto far_tag) {  // kFar: logits so low that e^a is 0, where 0 * -inf is not
      constexpr bool kFar = decltype(far_tag)::value;
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        u64 d = mul2(add2(pair(x[i], x[i + 1]), neg), scale);
        float a, b;
        unpair(d, a, b);
        if constexpr (kFar) {
          a = max_nan(a, -1000.f);
          b = max_nan(b, -1000.f);
          if constexpr (kChecked) {
            a = valid(i) ? a : -1000.f;
            b = valid(i + 1) ? b : -1000.f;
          }
          d = pair(a, b);
        }
        const u64 e = pair(lp_ex2(a), lp_ex2(b));
        s2 = add2(s2, e);
        w2 = fma2(e, d, w2);
      }
    };
    if (kChecked || __any_sync(0xffffffffu, low - mu < -600.f)) terms(std::true_type{});
    else terms(std::false_type{});
    float a, b;
    unpair(s2, a, b);
    sum.s += a + b;
    unpair(w2, a, b);
    sum.w += a + b;
    if (!kChecked && (end <= t || begin > t)) {
      const float bound = begin > t ? above : xt;
      u64 n2 = 0;  // counted as floats: the adds take the pipe that has room
#pragma unroll
      for (int i = 0; i < 16; i += 2) n2 = add2(n2, pair(at_least(x[i], bound), at_least(x[i + 1], bound)));
      unpair(n2, a, b);
      count += (int)(a + b);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (!kChecked || valid(i)) count += x[i] >= (index(i) < t ? xt : above) && index(i) != t;
    }
    if constexpr (TOP) {
      int taken = 16;
      if (first) {  // the lanes' maxima are the first list
        first = false;
#pragma unroll
        for (int i = 15; i >= 0; --i)
          if ((!kChecked || valid(i)) && x[i] == top) taken = i;
        list = sort32(taken < 16 ? entry_of(top, index(taken)) : 0ull, lane);
        raise(top_n, lane);
      }
      if (__any_sync(0xffffffffu, !(top < bar_value))) {
        uint32_t reach = 0;  // this lane's logits that may be among the best
#pragma unroll
        for (int i = 0; i < 16; ++i) reach |= (!kChecked || valid(i)) && !(x[i] < bar_value) ? 1u << i : 0u;
        reach &= ~(1u << taken);
        while (__any_sync(0xffffffffu, reach != 0)) {  // one logit a lane at a time
          const int i = reach ? __ffs(reach) - 1 : 0;
          float v = x[0];
#pragma unroll
          for (int j = 1; j < 16; ++j) v = j == i ? x[j] : v;  // registers have no index
          const u64 e = reach ? entry_of(v, index(i)) : 0;
          reach &= reach - 1;
          unsigned pass = __ballot_sync(0xffffffffu, e > bar);
          for (; pass; pass &= pass - 1) insert(__shfl_sync(0xffffffffu, e, __ffs(pass) - 1), lane);
          raise(top_n, lane);
        }
      }
    }
  }
};

CCUT_DEVICE float4 lp_remote4(uint32_t addr) {  // of another CTA of the cluster
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
CCUT_DEVICE u64 lp_remote(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

template <bool BF16, bool TOP>
__global__ void __launch_bounds__(kLpWarps * 32, 3) logprobs_kernel(LpArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ float bars[kLpWarps];
  __shared__ u64 lists[TOP ? kLpWarps : 1][TOP ? 32 : 1];
  __shared__ float4 stats[kLpWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows_per_cta = kLpWarps / a.wpr;
  const long long row = (long long)(blockIdx.x / a.ctas) * rows_per_cta + warp / a.wpr;
  const int cta = blockIdx.x % a.ctas, part = cta * a.wpr + warp % a.wpr, parts = a.ctas * a.wpr;
  const bool live = row < a.rows;
  LpWarp<TOP> st;
  st.row_bar = bars + warp / a.wpr * a.wpr;
  st.mine = &bars[warp];
  st.share = (a.top_n + a.wpr - 1) / a.wpr;
  if constexpr (TOP) {
    if (lane == 0) bars[warp] = -INFINITY;
    __syncthreads();
  }
  if (live) {
    constexpr int kVec = BF16 ? 8 : 4;  // logits per 16 bytes
    const char* base = static_cast<const char*>(a.x) + row * a.ld * (BF16 ? 2 : 4);
    const int t = a.tokens[row];
    const bool has = t >= 0 && t < a.vocab;
    const float xt = has ? logit<BF16>(base, t) : __int_as_float(0x7FFFFFFF);  // no token: nothing counts
    // the least float above xt: x > xt is x >= above (x_t = +inf: nothing is above, NaN compares false)
    const int kt = order_key(xt) + 1;
    const float above = isnan(xt) || xt == INFINITY ? __int_as_float(0x7FFFFFFF) : __int_as_float(kt < 0 ? kt ^ 0x7FFFFFFF : kt);
    const int lead = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / (BF16 ? 2 : 4));
    const int whole = (a.vocab - lead) / kLpRound;  // rounds of aligned 16-byte vectors
    const int r0 = (int)((long long)whole * part / parts), r1 = (int)((long long)whole * (part + 1) / parts);
    const uint4* src = reinterpret_cast<const uint4*>(base + (size_t)lead * (BF16 ? 2 : 4)) + lane;
    constexpr int kLoads = 16 / kVec;
    uint4 next[kLoads];
    auto fetch = [&](int r) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) next[j] = __ldcs(src + (size_t)r * (kLpRound / kVec) + j * 32);
    };
    if (r0 < r1) fetch(r0);
    for (int r = r0; r < r1; ++r) {
      float x[16];
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const uint32_t w[4] = {next[j].x, next[j].y, next[j].z, next[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (BF16) {
            x[j * 8 + 2 * e] = __uint_as_float(w[e] << 16);
            x[j * 8 + 2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
          } else {
            x[j * 4 + e] = __uint_as_float(w[e]);
          }
        }
      }
      if (r + 1 < r1) fetch(r + 1);
      if constexpr (TOP) st.look(a.wpr);
      const int begin = lead + r * kLpRound;
      st.template round<false>(
          x, [&](int i) { return begin + i / kVec * (32 * kVec) + lane * kVec + i % kVec; }, [](int) { return true; },
          begin, begin + kLpRound, t, xt, above, a.top_n, lane);
    }
    if (part == parts - 1) {  // what the vectors leave: the tail, then the head
      for (int side = 0; side < 2; ++side) {
        const int begin = side ? 0 : lead + whole * kLpRound, end = side ? lead : a.vocab;
        if (begin >= end) continue;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int v = begin + i * 32 + lane;
          x[i] = v < end ? logit<BF16>(base, v) : 0.f;
        }
        st.template round<true>(
            x, [&](int i) { return begin + i * 32 + lane; }, [&](int i) { return begin + i * 32 + lane < end; }, begin,
            end, t, xt, above, a.top_n, lane);
      }
    }
    if (has && isnan(xt)) {  // NaN is last in the order: everything else is before it, and NaN of lower index
      st.count = 0;
      const int v0 = part == 0 ? 0 : lead + r0 * kLpRound, v1 = part == parts - 1 ? a.vocab : lead + r1 * kLpRound;
      for (int v = v0 + lane; v < v1; v += 32) st.count += !isnan(logit<BF16>(base, v)) || v < t;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    LpSum y;
    y.m = __shfl_xor_sync(0xffffffffu, st.sum.m, o);
    y.s = __shfl_xor_sync(0xffffffffu, st.sum.s, o);
    y.w = __shfl_xor_sync(0xffffffffu, st.sum.w, o);
    st.sum.join(y);
  }
  int count = __reduce_add_sync(0xffffffffu, st.count);
  if (a.wpr > 1) {
    lp_tree<TOP>(st.sum, count, st.list, stats, lists, warp, lane, a.wpr);
  }
  if (a.ctas > 1) {  // warp w of the first CTA takes those of CTAs w and w + 8
    if (warp == 0) {
      if (lane == 0) stats[0] = make_float4(st.sum.m, st.sum.s, st.sum.w, __int_as_float(count));
      if constexpr (TOP) lists[0][lane] = st.list;
    }
    tc::cluster_sync();
    if (cta == 0) {
      st.sum = LpSum();
      count = 0;
      st.list = 0;
#pragma unroll
      for (int c = warp; c < kLpCluster; c += kLpWarps)
        if (c < a.ctas) {
          const float4 y = lp_remote4(tc::mapa(&stats[0], c));
          LpSum o;
          o.m = y.x, o.s = y.y, o.w = y.z;
          st.sum.join(o);
          count += __float_as_int(y.w);
          if constexpr (TOP) st.list = merge32(st.list, lp_remote(tc::mapa(&lists[0][lane], c)), lane);
        }
    }
    tc::cluster_sync();  // no CTA leaves while its state is read
    if (cta > 0) return;
    lp_tree<TOP>(st.sum, count, st.list, stats, lists, warp, lane, kLpWarps);
  }
  if (!live || warp % a.wpr) return;
  lp_finish<BF16, TOP>(a, row, st.sum, count, st.list, lane);
}

// Warps per row and CTAs per row.  At least 16 warps an SM, two rounds of logits or more for each.  With
// alternatives many rows take fewer warps each (2047 rows of 102400, top 20: 193 us with 8 warps a row, 171
// with 4, 176 with 1); without, eight keep the last round of CTAs short (136 us; 146 with 4).
static void lp_split(long long rows, int vocab, int top_n, int& wpr, int& ctas) {
  const long long want = 148LL * 16;
  wpr = top_n == 0 ? 8 : rows >= 2 * want ? 1 : rows >= want ? 2 : rows >= want / 2 ? 4 : 8;
  while (wpr > 1 && vocab < 2 * kLpRound * wpr) wpr /= 2;
  ctas = 1;
  if (rows * wpr < want) {
    long long c = want / (rows * wpr), most = vocab / (2 * kLpRound * wpr);
    if (c > most) c = most;
    while (ctas < kLpCluster && 2 * ctas <= c) ctas *= 2;  // above 1 only where wpr is 8: fewer leave no two rounds
  }
}

template <bool BF16, bool TOP>
static int run_logprobs(const LpArgs& a, cudaStream_t st) {
  const long long groups = (a.rows + kLpWarps / a.wpr - 1) / (kLpWarps / a.wpr);
  const dim3 grid((unsigned)(groups * a.ctas)), block(kLpWarps * 32);
  if (a.ctas == 1) return launch_k(logprobs_kernel<BF16, TOP>, grid, block, 0, st, a);
  static std::atomic<uint64_t> wide_set{0};  // devices on which clusters of more than 8 are allowed
  int rc = ensure_attribute(logprobs_kernel<BF16, TOP>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1, wide_set);
  if (rc) return rc;
  return launch_cluster(logprobs_kernel<BF16, TOP>, grid, block, 0, st, a.ctas, a);
}

}  // namespace ccut

using namespace ccut;

extern "C" {

int ccut_token_logprobs(const void* logits, int dtype, int rows, int vocab, long long ld, const int32_t* tokens,
                        int top_n, float* logprob, float* entropy, int32_t* rank, int32_t* top_ids,
                        float* top_logprobs, ccut_stream_t stream) {
  PdlScope pdl_scope(rows);
  if (dtype != CCUT_OUT_BF16 && dtype != CCUT_OUT_F32) return CCUT_ERR_INVALID;
  if (rows < 0 || vocab <= 0 || ld < vocab || top_n < 0 || top_n > vocab) return CCUT_ERR_INVALID;
  if (top_n > CCUT_MAX_TOP_LOGPROBS) return CCUT_ERR_UNSUPPORTED;
  if (rows == 0) return CCUT_OK;
  if (!logits || !tokens || !logprob || !entropy || !rank || (top_n > 0 && (!top_ids || !top_logprobs)))
    return CCUT_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == CCUT_OUT_BF16 ? 2 : 4)) return CCUT_ERR_INVALID;
  if (vocab > 2147483647 - 2 * kLpRound) return CCUT_ERR_UNSUPPORTED;
  LpArgs a{logits, vocab, ld, rows, tokens, top_n, 1, 1, logprob, entropy, rank, top_ids, top_logprobs};
  lp_split(rows, vocab, top_n, a.wpr, a.ctas);
  if (dtype == CCUT_OUT_BF16)
    return top_n ? run_logprobs<true, true>(a, stream) : run_logprobs<true, false>(a, stream);
  return top_n ? run_logprobs<false, true>(a, stream) : run_logprobs<false, false>(a, stream);
}

}  // extern "C"
