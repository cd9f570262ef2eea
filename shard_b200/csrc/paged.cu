// Writing to and reading from the paged 4-bit cache: append (rotary embedding, quantisation) and read-back.
//
// Both deal in vectors of 128 channels, four lanes to one (see paged.cuh): a warp takes eight vectors of one token,
// queries, keys and values alike, so that a token's cosines and sines are read once for the eight.
#include "paged.cuh"
#include "tcgen05.cuh"

namespace shard {

// ---- append --------------------------------------------------------------------------------------
// x' = rotation of x by the token's angle (pairs (c, c + 64); queries and keys), every product and sum rounded to
// fp32 on its own, so that the result is the formula's whatever the compiler would like to contract.  Then, for each
// 64 channels, held at +-32768:
//   s = fp16((max(x, 0) - min(x, 0)) * (1 / 15)) rounded to 7 significant bits (1 / 15 as an fp32 number),  z = rint(-min / s),
//   code = rint(x / s) + z, within 0 .. 15        (quotients, since 16-bit inputs do lie on the borders of codes)
//
// What bounds it: a warp waits for its rows, then computes (some 500 instructions) with nothing of its own in flight, and
// the 40 % of the warps that fit hide only a part of either from the other; in small calls, its chain of loads (tables, then
// angles).  8 191 tokens of 8 KV and 32 query heads, bf16 (101 MB in, 77 MB out): 40 us, 4.5 TB/s; 64 tokens: 5.6 us.  A
// warp takes eight vectors of a token rather than one vector: a maximum over 64 channels is two exchanges, not five, and
// angles are loaded once for the eight.
struct PagedAppendParams {
  ShardPaged c;
  const void *k, *v, *q;
  int64_t k_tok, k_head, v_tok, v_head, q_tok, q_head;   // in elements
  void* q_out;                                           // [rows][n_q][128]
  const float* rope;                                     // [rope_rows][64 cosines, 64 sines]
  int* status;
  int n_q, rows, rope_rows, chunks;
};

// (fminf and fmaxf drop a NaN, these keep it)
__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Parameter word of a half: its 64 channels are 16 in each of four neighbouring lanes.  Holds x at the limit.
__device__ __forceinline__ uint32_t pg_param(float (&x)[16]) {
  float lo = 0.f, hi = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = min_nan(max_nan(x[i], -PG_LIMIT), PG_LIMIT);
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (hi != hi) return 0x7e00u;
  const uint32_t bits = (__half_as_ushort(__float2half_rn(__fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f))) + 8u) & 0xfff0u;
  const float s = half_bits_to_float(bits);
  return bits | (s > 0.f ? (uint32_t)fminf(rintf(__fdiv_rn(-lo, s)), 15.f) : 0u);
}

// The codes of 16 channels of a half as two words: rint(x / s) + z within 0 .. 15, the quotient rounded to fp32.
// A division of its own for every value would be most of the kernel (and conversions to integers a good part of the
// rest), so the half's reciprocal r is taken once and the product y = x r corrected by what it leaves (Markstein, IBM J.
// Res. Dev. 34, 1990): y + (x - y s) r, the difference exact in one fused operation.  That is the rounded quotient
// itself: y is at most two last places off, so the correction is right to 2^-22 of a last place, and the quotient of
// 24 bits by the 7 of s is never nearer to the middle between two numbers than 2^-8 of one, nor on it.
__device__ __forceinline__ uint2 pg_codes(const float (&x)[16], float s, int z) {
  constexpr float MAGIC = 12582912.f;                    // 1.5 * 2^23: adding it rounds to whole numbers, in the low bits
  const bool any = s > 0.f;                              // (no scale, or NaN: the codes are the zero point)
  const float r = any ? __frcp_rn(s) : 0.f;
  if (!any) s = 0.f;
  const int bias = z - 0x4b400000;
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float y = __fmul_rn(x[i], r), q = fmaf(fmaf(-y, s, x[i]), r, y);
    w[i >> 3] += (uint32_t)min(max(__float_as_int(__fadd_rn(q, MAGIC)) + bias, 0), 15) << (4 * (i & 7));
  }
  return make_uint2(w[0], w[1]);
}

template <typename T>
__global__ void __launch_bounds__(128) paged_append_kernel(const __grid_constant__ PagedAppendParams p) {
  const int lane = threadIdx.x & 31, sub = lane & 3;
  griddep_launch();
  griddep_wait();
  const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int row = (int)(unit / (uint32_t)p.chunks), chunk = (int)(unit - (uint32_t)row * p.chunks);
  if (row >= p.rows) return;
  const int vec = 8 * chunk + (lane >> 2);               // queries, then keys, then values
  const int n_q = p.q ? p.n_q : 0, kv = vec - n_q;
  const bool is_q = vec < n_q, is_k = !is_q && kv < p.c.nkv, is_v = kv >= p.c.nkv && kv < 2 * p.c.nkv;
  // the vector's bytes are asked for before the row's sequence is known
  const T* src = is_q ? (const T*)p.q + row * p.q_tok + vec * p.q_head
               : is_k ? (const T*)p.k + row * p.k_tok + kv * p.k_head
                      : (const T*)p.v + row * p.v_tok + (kv - p.c.nkv) * p.v_head;
  uint4 raw[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      raw[h][e] = is_q || is_k || is_v ? *reinterpret_cast<const uint4*>(src + 64 * h + 16 * sub + 8 * e) : make_uint4(0u, 0u, 0u, 0u);
  const int b = paged_find_seq(p.c.cu, p.c.n_seqs, row, lane);
  if (b >= p.c.n_seqs) return;
  const PagedSeq seq = paged_seq(p.c, b, p.rows);
  if (row < seq.first || row >= seq.first + seq.n_new) return;
  const int pos = seq.pos0 + (row - seq.first);
  const bool placed = (unsigned)pos < (unsigned)p.rope_rows;
  if (!placed && chunk == 0 && lane == 0 && p.status) atomicOr(p.status, PG_BAD_POSITION);

  float x[2][16];                                        // [half][channel 16 sub + i]
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t w[4] = {raw[h][e].x, raw[h][e].y, raw[h][e].z, raw[h][e].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Pair<T>::get(w[i]);
        x[h][8 * e + 2 * i] = f.x;
        x[h][8 * e + 2 * i + 1] = f.y;
      }
    }
  if ((is_q || is_k) && placed) {
    const float4* cs = reinterpret_cast<const float4*>(p.rope + (int64_t)pos * HD) + 4 * sub;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 c4 = cs[e], s4 = cs[16 + e];
      const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = x[0][4 * e + i], d = x[1][4 * e + i];
        x[0][4 * e + i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(d, s[i]));
        x[1][4 * e + i] = __fadd_rn(__fmul_rn(d, c[i]), __fmul_rn(a, s[i]));
      }
    }
  }
  if (is_q) {
    T* dst = (T*)p.q_out + ((int64_t)row * p.n_q + vec) * HD;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = placed ? Pair<T>::put(x[h][8 * e + 2 * i], x[h][8 * e + 2 * i + 1]) : 0u;
        *reinterpret_cast<uint4*>(dst + 64 * h + 16 * sub + 8 * e) = make_uint4(w[0], w[1], w[2], w[3]);
      }
  }
  if (__all_sync(0xffffffffu, is_q)) return;
  uint32_t par[2];
  uint2 code[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    par[h] = pg_param(x[h]);
    code[h] = pg_codes(x[h], pg_scale(par[h]), (int)(par[h] & 15u));
  }
  if (!(is_k || is_v) || !placed) return;
  unsigned char* block = paged_block(p.c, b, pos, is_k ? kv : kv - p.c.nkv);
  if (!block) {
    if (sub == 0 && p.status) atomicOr(p.status, PG_BAD_PAGE);
    return;
  }
  const int t = pos % PG_BLOCK;
  *reinterpret_cast<uint4*>(block + (is_v ? PG_V : 0) + t * 64 + sub * 16) = make_uint4(code[0].x, code[1].x, code[0].y, code[1].y);
  if (sub == 0 && is_k) *reinterpret_cast<uint32_t*>(block + PG_KP + t * 4) = par[0] | (par[1] << 16);
  if (sub == 0 && is_v) {
    *reinterpret_cast<unsigned short*>(block + pg_vparam(t)) = (unsigned short)par[0];
    *reinterpret_cast<unsigned short*>(block + pg_vparam(t) + 8) = (unsigned short)par[1];
  }
}

// ---- read-back -----------------------------------------------------------------------------------
// A warp takes a row of the call, eight vectors at a time, and writes 32 bytes a lane (a whole sector): 79 % of what
// moves are the 16-bit numbers that come out.  Memory bounds it: eight sequences of up to 32 768 tokens, 8 KV heads (856
// MB moved): 143 us, 6.0 TB/s; 8 190 tokens: 10.7 us, most of which stays in L2.
struct PagedReadParams {
  ShardPaged c;
  void *k_out, *v_out;                                   // [rows][nkv][128]
  int* status;
  int rows;
};
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(128) paged_read_kernel(const __grid_constant__ PagedReadParams p) {
  const int lane = threadIdx.x & 31, sub = lane & 3;
  griddep_launch();
  griddep_wait();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int b = paged_find_seq(p.c.cu, p.c.n_seqs, row, lane);
  if (b >= p.c.n_seqs) return;
  const PagedSeq seq = paged_seq(p.c, b, p.rows);
  if (row < seq.first || row >= seq.first + seq.n_new) return;
  const int pos = seq.pos0 + (row - seq.first), t = pos & (PG_BLOCK - 1);
  const int64_t at = paged_block_offset(p.c, b, pos, 0), per_head = (int64_t)(p.c.page_size / PG_BLOCK) * PG_BYTES;
  if (at < 0 && lane == 0 && p.status) atomicOr(p.status, PG_BAD_PAGE);
#pragma unroll 2
  for (int vec = lane >> 2; vec < 2 * p.c.nkv; vec += 8) {
    const bool is_v = vec >= p.c.nkv;
    const int head = is_v ? vec - p.c.nkv : vec;
    uint4 code = make_uint4(0u, 0u, 0u, 0u);
    uint32_t par[2] = {0u, 0u};
    if (at >= 0) {
      const unsigned char* block = p.c.pool + at + head * per_head;
      code = *reinterpret_cast<const uint4*>(block + (is_v ? PG_V : 0) + t * 64 + sub * 16);
#pragma unroll
      for (int h = 0; h < 2; ++h) par[h] = *reinterpret_cast<const unsigned short*>(block + (is_v ? pg_vparam(t) + 8 * h : PG_KP + t * 4 + 2 * h));
    }
    T* dst = (T*)(is_v ? p.v_out : p.k_out) + ((int64_t)row * p.c.nkv + head) * HD + 16 * sub;
    const uint32_t w[2][2] = {{code.x, code.z}, {code.y, code.w}};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float s = pg_scale(par[h]), z = pg_zero(par[h]);
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v = w[h][i >> 2] >> (8 * (i & 3));
        o[i] = Pair<T>::put(((float)(v & 15u) - z) * s, ((float)((v >> 4) & 15u) - z) * s);
      }
      store32(dst + 64 * h, o);
    }
  }
}

// Launches CTAs of 128 threads that may be placed while the kernel in front still runs (they wait for it).
template <typename P>
static int launch_behind(void (*kernel)(P), unsigned grid, const P& p, void* stream) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(128);
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? SHARD_OK : (int)e;
}

}  // namespace shard

using namespace shard;

extern "C" size_t shard_b200_paged_page_bytes(int32_t nkv, int32_t page_size) {
  if (nkv < 1 || (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)) return 0;
  return (size_t)nkv * (page_size / PG_BLOCK) * PG_BYTES;
}

extern "C" int64_t shard_b200_paged_offset(const ShardPaged* cache_host, int32_t seq, int32_t pos, int32_t head) {
  if (paged_check(cache_host, 0) != SHARD_OK || seq < 0 || seq >= cache_host->n_seqs || head < 0 || head >= cache_host->nkv) return -1;
  return paged_block_offset(*cache_host, seq, pos, head);
}

extern "C" int shard_b200_paged_append(const ShardPaged* cache_host, const void* k, const void* v, const void* q, int64_t k_tok_stride,
                                       int64_t k_head_stride, int64_t v_tok_stride, int64_t v_head_stride, int64_t q_tok_stride,
                                       int64_t q_head_stride, int32_t n_q, int32_t rows, int32_t dtype, const float* rope,
                                       int32_t rope_rows, void* q_out, int* status_dev, void* stream) {
  const int rc = paged_check(cache_host, rows);
  if (rc != SHARD_OK) return rc;
  if (!k || !v || !rope || rope_rows < 0 || (q && (!q_out || n_q < 1 || n_q > 65536)) || (dtype != SHARD_F16 && dtype != SHARD_BF16))
    return SHARD_E_ARG;
  if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)rope) & 15) ||
      ((k_tok_stride | k_head_stride | v_tok_stride | v_head_stride | (q ? q_tok_stride | q_head_stride : 0)) & 7))
    return SHARD_E_ALIGN;
  if (rows == 0 || cache_host->n_seqs == 0) return SHARD_OK;
  PagedAppendParams p{*cache_host, k, v, q, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride, q_tok_stride, q_head_stride,
                      q_out, rope, status_dev, q ? n_q : 0, rows, rope_rows, 0};
  p.chunks = (p.n_q + 2 * p.c.nkv + 7) / 8;
  const int64_t grid = ((int64_t)rows * p.chunks + 3) / 4;
  if (grid > INT32_MAX / 4) return SHARD_E_TOO_LARGE;
  return launch_behind(dtype == SHARD_F16 ? paged_append_kernel<__half> : paged_append_kernel<__nv_bfloat16>, (unsigned)grid, p, stream);
}

extern "C" int shard_b200_paged_read_back(const ShardPaged* cache_host, int32_t rows, int32_t dtype, void* k_out, void* v_out,
                                          int* status_dev, void* stream) {
  const int rc = paged_check(cache_host, rows);
  if (rc != SHARD_OK) return rc;
  if (!k_out || !v_out || (dtype != SHARD_F16 && dtype != SHARD_BF16)) return SHARD_E_ARG;
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 31) return SHARD_E_ALIGN;
  if (rows == 0 || cache_host->n_seqs == 0) return SHARD_OK;
  PagedReadParams p{*cache_host, k_out, v_out, status_dev, rows};
  return launch_behind(dtype == SHARD_F16 ? paged_read_kernel<__half> : paged_read_kernel<__nv_bfloat16>, ((unsigned)rows + 3) / 4, p, stream);
}
