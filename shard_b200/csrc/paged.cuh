// The paged 4-bit cache: layout of its pages, and how a row of a call finds its sequence.
//
// Pool: [page][KV head][page_size / 16] blocks of 2176 bytes, a block = 16 consecutive tokens of one head:
//   0     codes of the keys, 64 bytes a token: the 8 channels 64 h + 8 g .. + 7 (half h, g < 8) are the nibbles of
//         the 32-bit word at 8 g + 4 h, lowest first
//   1024  codes of the values, the same
//   2048  parameters of the keys: 16-bit words [token][half]
//   2112  parameters of the values: 16-bit words [token % 8 / 2][half][token / 8][token % 2]
// A token's codes are one aligned 64-byte row, which four lanes read or write 16 bytes each: lane j has the
// channels 16 j .. 16 j + 15 of both halves, so the pairs (c, c + 64) that rotate together and half of what shares
// a parameter are its own.  Read as matrix fragments the same 16 bytes are the lane's share of eight k-steps.  The
// values' parameters lie as the lanes of a product over 16 tokens want them, two tokens to a word.
//
// A parameter belongs to 64 channels of a token: fp16 bits of a scale s with 7 significant bits, and in the four
// bits that leaves a zero point z.  A code stands for (code - z) * s.  Four bits times seven are eleven: every value
// of the cache is an fp16 number, so no kernel rounds when it unpacks, and 68 bytes hold a vector of 128 channels.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace shard {

constexpr int PG_BLOCK = 16;                  // tokens of a block
constexpr int PG_BYTES = SHARD_PAGED_BLOCK_BYTES;
constexpr int PG_V = 1024, PG_KP = 2048, PG_VP = 2112;
constexpr float PG_LIMIT = 32768.f;           // values beyond are held at it: no product of code and scale overflows fp16

enum { PG_BAD_PAGE = 1, PG_BAD_POSITION = 2, PG_BAD_COUNT = 4, PG_GAVE_UP = 8 };

// Byte of a token's first parameter word of the values; half 1 is 8 bytes behind.
__device__ __forceinline__ int pg_vparam(int t) { return PG_VP + (t % 8 / 2) * 16 + (t / 8) * 4 + (t % 2) * 2; }

struct PagedSeq {
  int first, n_new;   // rows first .. first + n_new - 1 of the call are this sequence's newest tokens
  int len, pos0;      // tokens it has with them (>= 0); position of the first one (may be negative: not a token then)
};

// (cu need not be well-formed: rows are cut to the call's, counts to what is there)
__device__ __forceinline__ PagedSeq paged_seq(const ShardPaged& c, int b, int rows) {
  PagedSeq s;
  s.first = min(max(c.cu[b], 0), rows);
  s.n_new = max(min(c.cu[b + 1], rows) - s.first, 0);
  s.len = max(c.lens[b], 0);
  s.pos0 = s.len - s.n_new;
  return s;
}

// The sequence of a row: how many entries cu[1 ..] are not above it, by a search in which each lane of the warp
// looks at one entry of 32 (one round trip to memory for 32 sequences, two for 1 000).  n_seqs if the row is behind
// the last one's.
__device__ __forceinline__ int paged_find_seq(const int32_t* __restrict__ cu, int n_seqs, int row, int lane) {
  int lo = 0, n = n_seqs;
  while (n > 0) {
    const int step = (n + 31) / 32, at = (lane + 1) * step;
    const bool below = at <= n && cu[lo + at] <= row;
    const int k = __popc(__ballot_sync(0xffffffffu, below));
    lo += k * step;
    n = min(step - 1, n - k * step);
  }
  return lo;
}

// Offset in the pool of the block that holds position `pos` of sequence b for one KV head, or -1 where the table has
// no page of the pool for it.
__host__ __device__ __forceinline__ int64_t paged_block_offset(const ShardPaged& c, int b, int pos, int head) {
  const int slot = pos / c.page_size;
  if (pos < 0 || slot >= c.table_width) return -1;
  const int page = c.page_table[b * c.table_stride + slot];
  if ((unsigned)page >= (unsigned)c.n_pages) return -1;
  const int64_t per_head = (int64_t)(c.page_size / PG_BLOCK) * PG_BYTES;
  return ((int64_t)page * c.nkv + head) * per_head + (pos % c.page_size) / PG_BLOCK * PG_BYTES;
}
__device__ __forceinline__ unsigned char* paged_block(const ShardPaged& c, int b, int pos, int head) {
  const int64_t at = paged_block_offset(c, b, pos, head);
  return at < 0 ? nullptr : c.pool + at;
}

__device__ __forceinline__ float half_bits_to_float(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
__device__ __forceinline__ float pg_scale(uint32_t word) { return half_bits_to_float(word & 0xfff0u); }
__device__ __forceinline__ float pg_zero(uint32_t word) { return (float)(word & 15u); }

template <typename T> struct Pair;            // two values of a 16-bit type in a register
template <> struct Pair<__half> {
  static __device__ __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ __half one(float a) { return __float2half_rn(a); }
};
template <> struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 get(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t put(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ __nv_bfloat16 one(float a) { return __float2bfloat16_rn(a); }
};

// What is wrong with a call's description, or SHARD_OK (host).
inline int paged_check(const ShardPaged* c, int rows) {
  if (!c || !c->pool || (!c->page_table && c->table_width > 0) || !c->cu || !c->lens || c->n_seqs < 0 || rows < 0 || c->nkv < 1 || c->n_pages < 0 ||
      c->table_width < 0 || c->table_stride < c->table_width)
    return SHARD_E_ARG;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return SHARD_E_ARG;
  if (c->n_seqs > SHARD_PAGED_MAX_SEQS || c->nkv > 1024 || (int64_t)c->table_width * c->page_size > (1 << 30)) return SHARD_E_ARG;
  if ((uintptr_t)c->pool & 15) return SHARD_E_ALIGN;
  return SHARD_OK;
}

}  // namespace shard
