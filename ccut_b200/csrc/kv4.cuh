// kv4.cuh -- the 4-bit kv cache format shared by its writer, its reader and the attention kernels.
//
// A cache row is one (slot, kv head, position): row = slot * slot_rows + head * max_len + position.
// Codes: head_dim / 2 bytes per row, byte j holds feature 2 j (low nibble) and 2 j + 1 (high nibble).
// Params: head_dim / 64 pairs (scale s, minimum m) of fp16 per row, one pair per group of 64 features;
// the value of code q is q s + m.  One pair per 64 features keeps the params at 4 of 36 bytes, and
// 64 features are four k16 steps of an MMA, so a group's scale can be applied to the fp32 product of
// the codes instead of to every code.
//
// Rounding: m = fp16(min) and s = fp16(fl32(max - m) * fl32(1/15)) to the nearest (two roundings of
// 2^-11; the codes are chosen with the rounded pair, so they only move the grid), q = the nearest of
// 0..15, ties to even.  Values beyond +-65504 saturate there, so s <= 8736 and q s + m <= 65536.
// A group that holds a NaN or an infinity gets s = m = NaN and reads back NaN.
#pragma once

#include "host.cuh"

namespace ccut {

constexpr int kKv4Group = 64;

// The value of code q under the pair (s, m): q * s has at most 15 significant bits, so the fma rounds once.
CCUT_DEVICE float kv4_value(uint32_t q, float s, float m) { return fmaf((float)q, s, m); }

// Two floats in a register pair, and the three-operand maximum.
typedef unsigned long long u64;
CCUT_DEVICE u64 pf_pair(float a, float b) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
CCUT_DEVICE void pf_unpair(u64 p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
CCUT_DEVICE u64 pf_add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
CCUT_DEVICE u64 pf_fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
CCUT_DEVICE u64 pf_mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
CCUT_DEVICE float pf_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Probabilities enter the second product as fp16, relative to a maximum that moves when a score passes it by 2^kKv4Lag
// and scaled by 2^kKv4Room: at most 2^15, with 11 bits down to 2^-25 (17 nats below the maximum) and nothing lost before
// 2^-36 (25 nats).  What a position without values (a sink) leaves to thousands of others is made of such small ones: unscaled,
// with a lag of 8, outputs were 1.5% off at 16 nats and zeros at 17.5.  The lag of 4 costs nothing (64 ragged
// caches 50.2 us with either, 4096 rows 148.5).
constexpr int kKv4Lag = 4, kKv4Room = 11;

// Host-side shape checks shared by the entry points.
inline bool kv4_shape_ok(int kv_heads, int head_dim, int max_len, long long slot_rows, int num_slots) {
  return kv_heads > 0 && (head_dim == 64 || head_dim == 128) && max_len > 0 && num_slots >= 0 &&
         slot_rows >= (long long)kv_heads * max_len;
}
inline bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

// A cache as the attention kernels read it.
struct Kv4Cache {
  const uint8_t* kc;
  const __half2* kp;
  const uint8_t* vc;
  const __half2* vp;
  int max_len;
  long long slot_rows;
};

// kv4_prefill.cu: query blocks of at least this many rows per kv head, whatever else.  Short-block / long-block kernel, 4
// kv heads, d = 128: 128 rows on one sequence of 8000 27.9 / 30.8 us, on eight of 4000 55 / 51; 160 rows 28 / 31 and
// 70 / 52 (d = 64, four of 4000: 27.0 / 26.6 and 30.7 / 26.9).  So one sequence would stay with the short blocks
// beyond 128 rows (10%) and a full machine would leave them before (8%): the limit lies between.  The short blocks
// also keep exact keys and values, and need no workspace for an unpacked cache.
constexpr int kKv4LongRows = 129;
bool kv4_prefill_fits(int batch, int heads, int kv_heads, int seq, int kv_len);
size_t kv4_prefill_workspace(int batch, int heads, int kv_heads, int seq, int kv_len, int head_dim);
int launch_kv4_prefill(const Kv4Cache& c, const uint16_t* q, const int32_t* slots, const int32_t* starts, int batch,
                       int heads, int kv_heads, int seq, int head_dim, int kv_len, int num_slots, float scale,
                       float softcap, void* out, bool out_bf16, void* workspace, int* status, cudaStream_t st);
long long kv4_wait_budget(long long cycles);  // of this thread's later launches; returns the one before

}  // namespace ccut
