// What the two kernels of the paged attention share: paged_attn.cu (few query rows to a sequence and KV head) and
// paged_tile.cu (many).
#pragma once

#include <climits>

#include "paged.cuh"
#include "tcgen05.cuh"

namespace shard {

// Sequences with more query rows to a KV head (new tokens times query heads of it) are paged_tile.cu's; the others too
// where, going by the sizes, all have more: paged_attn.cu's launches would find nothing to do.  64 sequences of 8 192
// tokens, 8 KV heads, paged_attn.cu / paged_tile.cu: 16 rows 298 / 513 us, 24 rows 439 / 514, 32 rows 620 / 535 (which cost
// the tiles the same, in four copies).  Up to 24 rows paged_attn.cu was faster at every length and number of sequences
// measured.  Of short sequences it is with more, too, so that rows alone put the border too low for them: 32 rows of 64
// sequences of 2 051 tokens 170 / 210 us, of one 15 / 26; 48 rows of one 16 / 27, of 64 247 / 220.
constexpr int PA_SHORT_ROWS = 24;

// A row's reference point is put PA_HEAD below its largest score so far, which then has the weight 2^7, and stays until
// a weight would pass 2^15: the two fp16 parts of a weight reach down to 2^-32 of the largest that way.
constexpr float PA_HEAD_LOG2 = 7.f, PA_MOST_LOG2 = 15.f;
constexpr float PA_NOTHING = -3e38f;                     // reference point before the first visible token
// A weight is 2 to the power of score * f - reference point, one fused operation, and what is scaled from one reference
// point to another is scaled by the difference of these very numbers: equal keys have equal weights, in whichever block,
// warp or piece they lie.  From 2^28 on no fp32 number is near enough to every product.  There different scores are 16 apart
// at least (as exponents), so a factor that makes them more changes nothing: f becomes the next power of two, and the
// product with the largest score is a number.
constexpr float PA_FAR = 268435456.f, PA_MOST_F = 8.5e37f;    // (2^126: the next power of two is one too)

// The tensor core cuts off what an fp32 accumulator has no bits for: some 2^-24 of a sum is lost with every product of 16
// tokens, always toward zero (131 072 tokens in one accumulator: 7e-4, more than an fp16 output's rounding).  So both
// kernels put an accumulator aside after 256 such products at most, and add up what they put aside in fp32 with
// rounding to nearest: 1.3e-5, whatever the length.  Putting it aside twice as often costs 3 % of the largest piece.

struct PagedAttnParams {
  ShardPaged c;
  const void* q;
  int64_t q_tok, q_head;
  void* out;                                             // [rows][n_q][128]
  float* lse;                                            // [rows][n_q] or null
  int* status;
  float* part;                                           // [2 grid][cols][132], and the split kernel's accumulators that are put aside
  int4* items;                                           // [grid] of the work that begins in a CTA's run and ends behind it
  float scale;
  int n_q, rows, max_new, ratio;
  int short_rows;                                        // sequences of up to that many rows are paged_attn.cu's
  int page_log2;                                         // blocks of a page: 1 << page_log2
  uint32_t ratio_mul, ratio_shift;                       // n / ratio = (n + high word of n * mul) >> shift for n < 2^31

  // (the hardware has no integer division: the compiler's takes some 200 cycles, and a row's head is a remainder)
  void set_ratio(int r) {
    ratio = r;
    ratio_shift = 0;
    while ((1u << ratio_shift) < (uint32_t)r) ++ratio_shift;
    ratio_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << ratio_shift) - (uint64_t)r)) / (uint64_t)r + 1);
  }
  __device__ __forceinline__ int over_ratio(int n) const { return (int)((__umulhi((uint32_t)n, ratio_mul) + (uint32_t)n) >> ratio_shift); }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float one_over(float power_of_two) { return __uint_as_float(0x7f000000u - __float_as_uint(power_of_two)); }
// The reference point moves to a largest score `most`: f and ref are the new ones (f0 the true f), the result is what sums
// so far have to be scaled by.
__device__ __forceinline__ float pa_move(float most, float f0, float& f, float& ref) {
  const float was = ref, was_f = f, near = fmaf(most, f0, -PA_HEAD_LOG2);
  f = fabsf(near) < PA_FAR ? f0 : __uint_as_float((__float_as_uint(f0) + 0x7fffffu) & 0x7f800000u);
  ref = fabsf(near) < PA_FAR ? near : most * f;
  return ex2(was_f == f ? was - ref : was_f == f0 ? -fmaf(most, f0, -was) : fmaf(was * one_over(was_f), f0, -ref));
}
// The reference point as others are to see it, of products with f0: a number m, and what sums have to be scaled by for it (1
// unless f is not f0; the rest of the largest product, while 2 to its power is a number of a sensible size).
__device__ __forceinline__ float pa_record(float ref, float f, float f0, float& m) {
  m = ref;
  if (f == f0) return 1.f;
  const float most = ref * one_over(f);
  m = most * f0;
  return fabsf(m) < 4.f * PA_FAR ? ex2(fmaf(most, f0, -m)) : 1.f;
}

// 1024 + the nibbles that `mask` leaves (16 times them from bits 4-7), in both halves
__device__ __forceinline__ uint32_t pa_1024(uint32_t x, uint32_t mask, uint32_t magic) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(magic));
  return d;
}

__device__ __forceinline__ int64_t pa_div(int64_t a, int64_t b) {    // (a 64-bit division takes hundreds of cycles)
  return a <= UINT32_MAX && b <= UINT32_MAX ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// Of two parameter words, those that are no numbers: all bits of their halves.
__device__ __forceinline__ uint32_t bad_words(uint32_t w) {
  return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}
// The first token of t, t + 1 (bad words `a`), t + 8, t + 9 (`b`) that is none.
__device__ __forceinline__ int first_bad(uint32_t a, uint32_t b, int t) {
  return a & 0xffffu ? t : a ? t + 1 : b & 0xffffu ? t + 8 : b ? t + 9 : INT_MAX;
}

// implemented in paged_tile.cu; needs paged_tile_bytes() of workspace
size_t paged_tile_bytes();
cudaError_t launch_paged_tile(const PagedAttnParams& p, bool bf16, void* workspace, cudaStream_t st);

}  // namespace shard
