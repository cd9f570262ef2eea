// Causal attention of the newest tokens of every sequence over its pages of the 4-bit cache.
//
//   s_t = scale * q . k_t,  o = sum_t exp(s_t) v_t / sum_t exp(s_t)   over t <= position of the row
//
// The work is a list of blocks (16 tokens of one KV head, for up to COLS query rows of it), sequence after sequence;
// every CTA takes an equal run of it, whatever the sequences' lengths, and its four warps take the blocks in turn.
// Where a run begins or ends inside a sequence's blocks, the CTA leaves a partial result (maximum, sum, accumulator per
// row), and paged_merge_kernel joins those in the list's order.
//
// A warp copies blocks (2 176 bytes) into a ring of its own, a group of two ahead, and multiplies with mma.sync m16n8k16:
//   scores   A = keys' codes, B = query.  A nibble in bits 6-9 of a half is the subnormal code * 2^-18, one in bits 2-5
//            a sixteenth of that (its query channel is taken 16 times): half a shift and a mask are all the unpacking
//            there is.  Not lower: the tensor core lines products up by their exponents, and a subnormal's is 2^-14
//            however few of its bits are set (nibbles in bits 0-3 and 4-7: scores of thousands were 2.5e-6 of
//            themselves off, now a tenth of that).  The query is scaled by a power of two into fp16's range.  s = sum over halves of
//            scale_h * (codes . q - z_h * sum(q)), the latter in fp32.
//   output   A = values (channels x tokens), B = weights.  Pairs of tokens are one byte permutation of their words;
//            (1024 + code) - (1024 + z) and the product with the scale are exact in fp16.  A weight is two fp16 parts
//            (22 bits, see PA_HEAD_LOG2): up to four rows fill a tile's eight columns with them, so that they are free there.
//
// What bounds it: instructions.  A block is some 375 of a warp's (half of them masks, shifts and fp16 arithmetic that
// unpack) and takes a scheduler 600 cycles with three warps to choose from; the bytes would come 1.7 times as fast.  64
// sequences of up to 8 192 tokens, 8 KV heads, 4 query heads to each (433 MB): 117 us, 3.7 TB/s; one of 131 072 (143 MB):
// 45 us, 3.2 TB/s.  Fixed part of a launch, some 10 000 cycles: adding the list up 2 000, the query 2 000, the first
// blocks 1 300, joining the warps; then the launch that joins the CTAs, 3 to 5 us.
#include <atomic>
#include <type_traits>

#include "paged_attn.cuh"

namespace shard {

constexpr int PA_WARPS = 4;                              // (5, 7, 8: slower)
constexpr int PA_CTAS = 3;                               // per SM, 168 registers a thread (4 and 128: spills, 135 us where this took 124)
constexpr int PA_GROUP = 2;                              // blocks that a warp takes at a time (4: no room in registers, slower)
constexpr int PA_STAGES = 2;                             // such groups in its ring (3: the same)
constexpr int PA_HOLD = 64;                              // turns of a warp whose products add up in its accumulators (see paged_attn.cuh)
constexpr int PA_MIN_BLOCKS = 4;                         // of a CTA's run: one for each warp
constexpr uint32_t PA_NO_BLOCK = 0xffffffffu;
constexpr int PA_HELD = 32 * 36;                         // numbers in a warp's accumulators, and where they count from

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
// What a sequence adds to the list: its blocks, and how many times COLS rows of a KV head it has.
struct PagedShare {
  int blocks, groups;
};
template <int COLS>
__device__ __forceinline__ PagedShare paged_share(const PagedAttnParams& p, const PagedSeq& s) {
  const int n = min(s.len, p.c.table_width * p.c.page_size);
  if (s.n_new > p.max_new || s.n_new * p.ratio > p.short_rows) return {0, 0};
  // (a sequence that has rows and no token still has one block, which shows its rows nothing)
  return {max((n + PG_BLOCK - 1) / PG_BLOCK, 1), (s.n_new * p.ratio + COLS - 1) / COLS};
}

// Blocks lie in a warp's ring in shared memory.  A copy there has the 16-byte pieces of
// every 128 bytes of codes (two tokens) exchanged, by twice the pair's number, so that neither the rows of keys that
// eight lanes read at once nor the values of four pairs of tokens that sixteen lanes read meet in a bank.
__device__ __forceinline__ uint32_t pa_piece(int i) { return (uint32_t)((i >> 3) * 128 + ((i & 7) ^ (2 * ((i >> 3) & 3))) * 16); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// COLS: query rows to a tile.  4: the tile's other four columns carry the same rows again, and then the low parts of
// their weights.  8: two products for the two parts.  Chosen by a sequence's largest number of rows: four rows in eight
// columns take 157 us where four take 147 (64 sequences of 8 192 tokens, 8 KV heads), eight rows 158 and 278.
template <typename T, int COLS>
__global__ void __launch_bounds__(32 * PA_WARPS, PA_CTAS) paged_split_kernel(const __grid_constant__ PagedAttnParams p) {
  extern __shared__ __align__(16) unsigned char pa_smem[];
  // a ring of blocks for each warp, which holds its result for the others at the end of a piece of work
  constexpr int RING = PA_STAGES * PA_GROUP * PG_BYTES;
  static_assert(COLS * PART * 4 <= RING, "a warp's result fits its ring");
  auto state = [&](int w, int c) { return reinterpret_cast<float*>(pa_smem + w * RING) + c * PART; };
  int64_t* before = reinterpret_cast<int64_t*>(pa_smem + PA_WARPS * RING);   // [n_seqs + 1] blocks before a sequence's
  __shared__ int64_t warp_sum[PA_WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
  griddep_launch();
  griddep_wait();

  {  // the list: every CTA adds it up for itself
    const int n = p.c.n_seqs, each = (n + 32 * PA_WARPS - 1) / (32 * PA_WARPS), b0 = min(tid * each, n), b1 = min(b0 + each, n);
    int64_t sum = 0;
    for (int b = b0; b < b1; ++b) {
      const PagedSeq s = paged_seq(p.c, b, p.rows);
      const PagedShare w = paged_share<COLS>(p, s);
      before[b] = sum;
      sum += (int64_t)w.blocks * w.groups * p.c.nkv;
      if (blockIdx.x == 0 && p.status && s.n_new > 0) {
        if (s.n_new > p.max_new) atomicOr(p.status, PG_BAD_COUNT);
        else if (s.len > p.c.table_width * p.c.page_size) atomicOr(p.status, PG_BAD_PAGE);
      }
    }
    int64_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int64_t base = incl - sum, all = 0;
#pragma unroll
    for (int w = 0; w < PA_WARPS; ++w) {
      if (w < warp) base += warp_sum[w];
      all += warp_sum[w];
    }
    for (int b = b0; b < b1; ++b) before[b] += base;
    if (tid == 0) before[n] = all;
    __syncthreads();
  }
  const int64_t total = before[p.c.n_seqs];
  const int64_t ctas = min((int64_t)gridDim.x, (total + PA_MIN_BLOCKS - 1) / PA_MIN_BLOCKS);
  if (tid == 0) p.items[blockIdx.x] = make_int4(0, 0, 0, 0);
  if (blockIdx.x >= ctas) return;
  // runs of `each` blocks, the first `more` of them one longer
  const int64_t each = pa_div(total, ctas), more = total - each * ctas;
  const int64_t begin = each * blockIdx.x + min((int64_t)blockIdx.x, more), end = begin + each + (blockIdx.x < more);
  int b = 0;
  {
    int lo = 0, hi = p.c.n_seqs;                         // the last sequence that does not begin behind `begin`
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= begin) lo = mid; else hi = mid;
    }
    b = lo;
  }
  for (int64_t at = begin; at < end;) {
    while (before[b + 1] <= at) ++b;
    const PagedSeq seq = paged_seq(p.c, b, p.rows);
    const PagedShare share = paged_share<COLS>(p, seq);
    const int64_t in_seq = at - before[b];
    const int unit = (int)pa_div(in_seq, share.blocks), blk0 = (int)(in_seq - (int64_t)unit * share.blocks);
    const int blk1 = (int)min((int64_t)share.blocks, blk0 + (end - at));
    const int kv = unit / share.groups, col0 = (unit - kv * share.groups) * COLS;
    const int cols = min(COLS, seq.n_new * p.ratio - col0);
    const int room = min(seq.len, p.c.table_width * p.c.page_size);

    uint32_t magic;                                      // 1024 in both halves, kept in a register: one instruction masks and adds it
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));

    // ---- the blocks, a group a turn: looked up two turns ahead, copied one ahead (the first before the query is looked at)
    const int32_t* table = p.c.page_table + b * p.c.table_stride;
    const int group = min(PA_GROUP, (blk1 - blk0 + PA_WARPS - 1) / PA_WARPS);      // (little work: all warps have some)
    const uint32_t ring = smem_u32(pa_smem) + warp * RING, k_at = ring + pa_piece(lane), par_at = ring + PG_KP;
    const uint32_t v_at[2] = {ring + PG_V + j * 128 + ((g >> 1) ^ (2 * j)) * 16 + (g & 1) * 8,
                              ring + PG_V + j * 128 + ((4 + (g >> 1)) ^ (2 * j)) * 16 + (g & 1) * 8};
    // lane i: where in the pool block `first` + i is, in blocks, or PA_NO_BLOCK where there is none
    auto look_up = [&](int first) {
      const int blk = first + (lane & (PA_GROUP - 1));
      uint32_t at_block = PA_NO_BLOCK;
      if ((lane & (PA_GROUP - 1)) < group && blk < blk1 && blk * PG_BLOCK < room) {
        const int page = table[blk >> p.page_log2];
        if ((unsigned)page < (unsigned)p.c.n_pages) at_block = (((uint32_t)page * p.c.nkv + kv) << p.page_log2) + (blk & ((1 << p.page_log2) - 1));
      }
      return at_block;
    };
    auto fetch = [&](uint32_t where, int slot) {         // (a block that is not there is not fetched: nothing of it is counted)
#pragma unroll
      for (int i = 0; i < PA_GROUP; ++i) {
        const uint32_t at_block = __shfl_sync(0xffffffffu, where, i);
        if (at_block != PA_NO_BLOCK) {
          const unsigned char* src = p.c.pool + (uint64_t)at_block * PG_BYTES + lane * 16;
          const uint32_t to = (slot * PA_GROUP + i) * PG_BYTES;
#pragma unroll
          for (int k = 0; k < 4; ++k) cp_async16(k_at + to + 512 * k, src + 512 * k);
          if (lane < 8) cp_async16(par_at + to + lane * 16, src + PG_KP);
        }
      }
      cp_async_commit();
      return __ballot_sync(0xffffffffu, where != PA_NO_BLOCK) & ((1u << PA_GROUP) - 1);
    };
    const int step = group * PA_WARPS;
    int first = blk0 + warp * group, slot = 0;
    uint32_t there = fetch(look_up(first), 0), next = look_up(first + step);

    // ---- query: column `g` of the tile, and what the lane's two score columns need to know
    uint32_t q[16], qsum;                                // (qsum: part j of -sum(q) of both halves)
    float f0[2], f[2];                                   // what a score is times for the exponent of 2
    int vis[2], vis_min;
    {
      const int col = COLS == 4 ? g & 3 : g, cc = col0 + col, tok = p.over_ratio(cc), head = kv * p.ratio + cc - tok * p.ratio;
      float x[2][16], top = 0.f;
      const T* src = (const T*)p.q + (int64_t)(seq.first + tok) * p.q_tok + head * p.q_head + 16 * j;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint4 u = make_uint4(0u, 0u, 0u, 0u);
          if (col < cols) u = *reinterpret_cast<const uint4*>(src + 64 * h + 8 * e);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 v = Pair<T>::get(w[i]);
            x[h][8 * e + 2 * i] = v.x;
            x[h][8 * e + 2 * i + 1] = v.y;
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // largest channel to 2^9 .. 2^10, with the sign of `scale`; a query of zeros, or one that is not finite, stays as it is
      const int ex = (int)(__float_as_uint(top) >> 23), up = top == 0.f || ex == 255 ? 127 : min(263 - ex, 250);
      const float by = p.scale == 0.f ? 0.f : copysignf(__uint_as_float((uint32_t)up << 23), p.scale), back = __uint_as_float((uint32_t)(254 - up) << 23);
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float v = __half2float(__float2half_rn(x[h][8 * e + i] * by));
            sum[h] += v;
            x[h][8 * e + i] = v;
          }
          const float* y = &x[h][8 * e];
          uint32_t* r = &q[8 * h + 4 * e];
          r[0] = pack_half2(y[0] * 16.f, y[4] * 16.f);
          r[1] = pack_half2(y[2] * 16.f, y[6] * 16.f);
          r[2] = pack_half2(y[1], y[5]);
          r[3] = pack_half2(y[3], y[7]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);   // (64 times less than 2^10: within fp16)
      }
      {  // four fp16 numbers whose sum is the fp32 one: lane j's is row 2 j (half 1: 2 j + 1) of a product with z
        __half part[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float rest = -sum[h];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __half top_part = __float2half_rn(rest);
            if (i == j) part[h] = top_part;
            rest -= __half2float(top_part);
          }
        }
        qsum = as_u32(__halves2half2(part[0], part[1]));
      }
      // (held: of bf16 queries from 2^120 on the weights are 0 and 1 all the same)
      const float factor = p.scale == 0.f ? 1.f : fminf(fmaxf(back * (262144.f * fabsf(p.scale) * LOG2E), 1e-37f), PA_MOST_F);
      const int see = col < cols ? min(max(seq.pos0 + tok + 1, 0), room) : room;   // (columns without a row hide nothing)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = 4 * (2 * j + c);
        f0[c] = f[c] = __shfl_sync(0xffffffffu, factor, from);
        vis[c] = __shfl_sync(0xffffffffu, see, from);
      }
      vis_min = (int)__reduce_min_sync(0xffffffffu, (uint32_t)see);
    }

    // ref: reference point; lim: how far above it a score may be (nothing yet: any score moves it)
    float o[8][4], ref[2] = {0.f, 0.f}, lim[2] = {PA_NOTHING, PA_NOTHING}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    // (FULL: a whole group, without a branch between its blocks, so that their instructions mix)
    auto turn = [&](auto full) {
      constexpr bool FULL = decltype(full)::value;
      cp_async_wait<0>();
      __syncwarp();                                      // all lanes' pieces have landed, and all are done with the group before
      const uint32_t here = there;
      there = fetch(next, slot ^ 1);
      next = look_up(first + 2 * step);
      const uint32_t off = slot * (PA_GROUP * PG_BYTES);

      // scores of rows g, g + 8 (tokens) and columns 2 j, 2 j + 1
      float s[PA_GROUP][4];
#pragma unroll
      for (int i = 0; i < PA_GROUP; ++i) {
        if (!FULL && i >= group) {
          s[i][0] = s[i][1] = s[i][2] = s[i][3] = neg_inf();
          continue;
        }
        const uint32_t o_ = off + i * PG_BYTES;
        const uint4 k0 = lds128(k_at + o_), k1 = lds128(k_at + o_ + 512);   // 32 channels of tokens g and g + 8
        const uint32_t kp0 = lds32(par_at + o_ + g * 4), kp1 = lds32(par_at + o_ + 32 + g * 4);
        const uint32_t kw[2][2][2] = {{{k0.x, k0.z}, {k1.x, k1.z}}, {{k0.y, k0.w}, {k1.y, k1.w}}};
        float half[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t mz = h ? 0x03c00000u : 0x000003c0u;
          float d[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};   // channels 0, 2, 4, 6 of eight; 1, 3, 5, 7
          mma_16816(d[1], (kp0 << 6) & mz, (kp1 << 6) & mz, 0u, 0u, qsum, 0u);   // -z sum(q)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t a = kw[h][0][u] << 2, c = kw[h][1][u] << 2, a2 = kw[h][0][u] >> 6, c2 = kw[h][1][u] >> 6;
            const uint32_t* r = &q[8 * h + 4 * u];
            mma_16816(d[0], a & 0x003c003cu, c & 0x003c003cu, a2 & 0x003c003cu, c2 & 0x003c003cu, r[0], r[1]);
            mma_16816(d[1], a & 0x03c003c0u, c & 0x03c003c0u, a2 & 0x03c003c0u, c2 & 0x03c003c0u, r[2], r[3]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) half[h][k] = d[0][k] + d[1][k];
        }
        const float2 s0 = __half22float2(as_half2(kp0 & 0xfff0fff0u)), s1 = __half22float2(as_half2(kp1 & 0xfff0fff0u));
#pragma unroll
        for (int k = 0; k < 4; ++k)
          s[i][k] = fmaf(k < 2 ? s0.y : s1.y, half[1][k], (k < 2 ? s0.x : s1.x) * half[0][k]);
      }
      const int t0 = first * PG_BLOCK;
      const int blocks = FULL ? PA_GROUP : group;
      const bool edge = t0 + blocks * PG_BLOCK > vis_min || here != (1u << blocks) - 1;
      if (edge) {
#pragma unroll
        for (int i = 0; i < PA_GROUP; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (!((here >> i) & 1) || t0 + PG_BLOCK * i + g + 8 * (k >> 1) >= vis[k & 1]) s[i][k] = neg_inf();
        if (lane < group && !((here >> lane) & 1) && first + lane < blk1 && t0 + PG_BLOCK * lane < room && p.status)
          atomicOr(p.status, PG_BAD_PAGE);
      }
      float most[2] = {fmaxf(s[0][0], s[0][2]), fmaxf(s[0][1], s[0][3])};
#pragma unroll
      for (int i = 1; i < PA_GROUP; ++i) {
        most[0] = fmaxf(most[0], fmaxf(s[i][0], s[i][2]));
        most[1] = fmaxf(most[1], fmaxf(s[i][1], s[i][3]));
      }
      if (__any_sync(0xffffffffu, fmaf(most[0], f[0], -ref[0]) > lim[0] || fmaf(most[1], f[1], -ref[1]) > lim[1])) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) most[c] = fmaxf(most[c], __shfl_xor_sync(0xffffffffu, most[c], d));
          if (fmaf(most[c], f[c], -ref[c]) > lim[c]) {   // (the same for all lanes of a column)
            float alpha = pa_move(most[c], f0[c], f[c], ref[c]);
            if (lim[c] != PA_MOST_LOG2) alpha = 0.f;
            lim[c] = PA_MOST_LOG2;
            l[c] *= alpha;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              o[i][c] *= alpha;
              o[i][2 + c] *= alpha;
            }
          }
        }
      }

#pragma unroll
      for (int i = 0; i < PA_GROUP; ++i) {
        if (!FULL && i >= group) continue;
        const uint32_t o_ = off + i * PG_BYTES;
        float w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = ex2(fmaf(s[i][k], f[k & 1], -ref[k & 1]));
        l[0] += w[0] + w[2];
        l[1] += w[1] + w[3];
        // weights as two fp16 parts, transposed: tokens 2 j, 2 j + 1 (and 8 on) of column g
        uint32_t hi0 = pack_half2(w[0], w[1]), hi1 = pack_half2(w[2], w[3]), lo0, lo1;
        {
          const float2 r0 = __half22float2(as_half2(hi0)), r1 = __half22float2(as_half2(hi1));
          lo0 = pack_half2(w[0] - r0.x, w[1] - r0.y);
          lo1 = pack_half2(w[2] - r1.x, w[3] - r1.y);
        }
        if (COLS == 4 && j >= 2) { hi0 = lo0; hi1 = lo1; }
        const uint32_t b0 = movmatrix(hi0), b1 = movmatrix(hi1);
        const uint32_t c0 = COLS == 8 ? movmatrix(lo0) : 0u, c1 = COLS == 8 ? movmatrix(lo1) : 0u;

        uint4 vp = lds128(par_at + o_ + 64 + j * 16);    // parameters: (half 0: two tokens, two tokens), half 1
        if (edge) {
          // 0 * NaN is not 0: values of tokens that nobody sees may have any parameters,
          const int at_block = t0 + PG_BLOCK * i, left = (here >> i) & 1 ? room - at_block : 0;
          const uint32_t m0 = (2 * j < left ? 0xffffu : 0u) | (2 * j + 1 < left ? 0xffff0000u : 0u);
          const uint32_t m1 = (2 * j + 8 < left ? 0xffffu : 0u) | (2 * j + 9 < left ? 0xffff0000u : 0u);
          vp.x &= m0; vp.y &= m1; vp.z &= m0; vp.w &= m1;
          // and those that only some rows see reach these without the product
          const uint32_t b0_ = bad_words(vp.x), b1_ = bad_words(vp.y), b2_ = bad_words(vp.z), b3_ = bad_words(vp.w);
          if (__any_sync(0xffffffffu, b0_ | b1_ | b2_ | b3_)) {
            const int first0 = (int)__reduce_min_sync(0xffffffffu, (uint32_t)first_bad(b0_, b1_, at_block + 2 * j));
            const int first1 = (int)__reduce_min_sync(0xffffffffu, (uint32_t)first_bad(b2_, b3_, at_block + 2 * j));
            vp.x &= ~b0_; vp.y &= ~b1_; vp.z &= ~b2_; vp.w &= ~b3_;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int u = 0; u < 8; ++u)
                if ((u < 4 ? first0 : first1) < vis[c]) o[u][c] = o[u][2 + c] = __uint_as_float(0x7fffffffu);
          }
        }
        uint2 v[4];                                      // channels 8 g .. of both halves, tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = lds64(v_at[k & 1] + o_ + 512 * (k >> 1));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t x[2][2];                              // [pair of tokens][channels 0-3, 4-7 of the lane's eight]
          __half2 sc[2], sc16[2], ze[2], ze16[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint32_t a = h ? v[2 * t].y : v[2 * t].x, c = h ? v[2 * t + 1].y : v[2 * t + 1].x;
            x[t][0] = __byte_perm(a, c, 0x5410);
            x[t][1] = __byte_perm(a, c, 0x7632);
            const uint32_t par = h ? (t ? vp.w : vp.z) : (t ? vp.y : vp.x);
            sc[t] = as_half2(par & 0xfff0fff0u);
            sc16[t] = __hmul2(sc[t], __float2half2_rn(0.0625f));   // (exact: a scale's last four bits are 0)
            ze[t] = as_half2(pa_1024(par, 0x000f000fu, magic));
            ze16[t] = __hfma2(ze[t], __float2half2_rn(16.f), __float2half2_rn(-15360.f));   // 1024 + 16 z
          }
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t y0 = e ? x[0][u] >> 8 : x[0][u], y1 = e ? x[1][u] >> 8 : x[1][u];
              const uint32_t a0 = as_u32(__hmul2(__hsub2(as_half2(pa_1024(y0, 0x000f000fu, magic)), ze[0]), sc[0]));
              const uint32_t a1 = as_u32(__hmul2(__hsub2(as_half2(pa_1024(y0, 0x00f000f0u, magic)), ze16[0]), sc16[0]));
              const uint32_t a2 = as_u32(__hmul2(__hsub2(as_half2(pa_1024(y1, 0x000f000fu, magic)), ze[1]), sc[1]));
              const uint32_t a3 = as_u32(__hmul2(__hsub2(as_half2(pa_1024(y1, 0x00f000f0u, magic)), ze16[1]), sc16[1]));
              float (&d)[4] = o[4 * h + 2 * u + e];
              mma_16816(d, a0, a1, a2, a3, b0, b1);
              if (COLS == 8) mma_16816(d, a0, a1, a2, a3, c0, c1);
            }
        }
      }
    };
    // What the accumulators had before their last PA_HOLD turns waits in memory, with its reference points.
    float4* held = reinterpret_cast<float4*>(p.part + (int64_t)2 * gridDim.x * COLS * PART + (blockIdx.x * PA_WARPS + warp) * PA_HELD) + lane;
    const int hold = PA_HOLD * step, first_hold = first + hold;
    auto add_held = [&]() {
      const float4 at = held[8 * 32];
      float m[2], by[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float scale = pa_record(ref[c], f[c], f0[c], m[c]);
        by[c] = ex2((c ? at.y : at.x) - m[c]) / scale;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 h = held[i * 32];
        o[i][0] = fmaf(h.x, by[0], o[i][0]);
        o[i][1] = fmaf(h.y, by[1], o[i][1]);
        o[i][2] = fmaf(h.z, by[0], o[i][2]);
        o[i][3] = fmaf(h.w, by[1], o[i][3]);
      }
    };
#pragma unroll 1
    for (int next_hold = first_hold; first < blk1; first += step, slot ^= 1) {
      if (first == next_hold) {
        if (first != first_hold) add_held();
        next_hold += hold;
        float m[2], by[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) by[c] = pa_record(ref[c], f[c], f0[c], m[c]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          held[i * 32] = make_float4(o[i][0] * by[0], o[i][1] * by[1], o[i][2] * by[0], o[i][3] * by[1]);
          o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        }
        held[8 * 32] = make_float4(lim[0] == PA_MOST_LOG2 ? m[0] : PA_NOTHING, lim[1] == PA_MOST_LOG2 ? m[1] : PA_NOTHING, 0.f, 0.f);
      }
      if (group == PA_GROUP) turn(std::true_type());
      else turn(std::false_type());
    }
    if (first > first_hold) add_held();
    cp_async_wait<0>();
    __syncwarp();

    // ---- the four warps' states become one
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[c] += __shfl_xor_sync(0xffffffffu, l[c], d);
    if (COLS == 4) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][k] += __shfl_xor_sync(0xffffffffu, o[i][k], 2);
    }
    if (COLS == 8 || j < 2) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* rec = state(warp, 2 * j + c);
        float m;
        const float by = pa_record(ref[c], f[c], f0[c], m);
        if (g == 0) *reinterpret_cast<float2*>(rec) = make_float2(lim[c] == PA_MOST_LOG2 ? m : PA_NOTHING, l[c] * by);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float (&e0)[4] = o[4 * h + 2 * u], (&e1)[4] = o[4 * h + 2 * u + 1];
            *reinterpret_cast<float4*>(rec + 4 + 64 * h + 8 * g + 4 * u) = make_float4(e0[c] * by, e0[2 + c] * by, e1[c] * by, e1[2 + c] * by);
          }
      }
    }
    __syncthreads();
    const bool whole = blk0 == 0 && blk1 == share.blocks;
    // (a run has at most two pieces of work that others share: the one it begins in and the one it ends in)
    float* part = p.part + (2 * (int64_t)blockIdx.x + (at == begin ? 0 : 1)) * COLS * PART;
    for (int c = warp; c < cols; c += PA_WARPS) {
      float ms[PA_WARPS], top = PA_NOTHING, sum = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        ms[w] = state(w, c)[0];
        top = fmaxf(top, ms[w]);
      }
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        const float* rec = state(w, c);
        const float by = ex2(ms[w] - top);
        const float4 v = *reinterpret_cast<const float4*>(rec + 4 + 4 * lane);
        sum = fmaf(rec[1], by, sum);
        a.x = fmaf(v.x, by, a.x);
        a.y = fmaf(v.y, by, a.y);
        a.z = fmaf(v.z, by, a.z);
        a.w = fmaf(v.w, by, a.w);
      }
      if (whole) {
        const int cc = col0 + c, tok = p.over_ratio(cc), head = kv * p.ratio + cc - tok * p.ratio;
        const int64_t row = (int64_t)(seq.first + tok) * p.n_q + head;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>((T*)p.out + row * HD + 4 * lane) = make_uint2(Pair<T>::put(a.x * inv, a.y * inv), Pair<T>::put(a.z * inv, a.w * inv));
        if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? neg_inf() : (top + log2f(sum)) * LN2;
      } else {
        float* rec = part + c * PART;
        if (lane == 0) *reinterpret_cast<float4*>(rec) = make_float4(top, sum, 0.f, 0.f);
        *reinterpret_cast<float4*>(rec + 4 + 4 * lane) = a;
      }
    }
    if (tid == 0 && blk0 == 0 && !whole) {
      // the work begins here and goes on in the next CTAs' runs
      const int64_t stop = at + share.blocks - 1;        // its last block, and whose run that is in
      const int last = (int)(stop < (each + 1) * more ? pa_div(stop, each + 1) : more + pa_div(stop - (each + 1) * more, each));
      p.items[blockIdx.x] = make_int4(b + 1, unit, last - (int)blockIdx.x + 1, at == begin ? 0 : 1);
    }
    at += blk1 - blk0;
    __syncthreads();
  }
}

// Joins the pieces of the work that begins in a CTA's run and ends behind it, always in the same order.  A CTA looks
// after PM_RUNS runs: work in up to PM_DEPTH pieces takes a warp a row, all of them in flight at once; work in more,
// as of one long sequence, takes all warps.  (With 8 columns a block has 1 024 threads of 64 registers, and 36 bytes spill.)
constexpr int PM_RUNS = 4, PM_DEPTH = 8;
template <typename T, int COLS>
__global__ void __launch_bounds__(32 * COLS * PM_RUNS) paged_merge_kernel(const __grid_constant__ PagedAttnParams p, int runs) {
  __shared__ __align__(16) float acc_s[PM_RUNS][COLS][PART];
  __shared__ int4 items[PM_RUNS];
  griddep_launch();
  griddep_wait();
  const int run0 = blockIdx.x * PM_RUNS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = warp % COLS, w = warp / COLS;
  if (threadIdx.x < PM_RUNS) items[threadIdx.x] = run0 + (int)threadIdx.x < runs ? p.items[run0 + threadIdx.x] : make_int4(0, 0, 0, 0);
  __syncthreads();
  float top, sum;
  float4 a;
  auto add = [&](float m, float l, float4 v) {
    const float now = fmaxf(top, m), old = ex2(top - now), by = ex2(m - now);
    top = now;
    sum = fmaf(l, by, sum * old);
    a.x = fmaf(v.x, by, a.x * old);
    a.y = fmaf(v.y, by, a.y * old);
    a.z = fmaf(v.z, by, a.z * old);
    a.w = fmaf(v.w, by, a.w * old);
  };
  // every `stride`-th piece from `begin` on
  auto gather = [&](int run, int4 item, int begin, int stride) {
    const float* first = p.part + ((2 * (int64_t)run + item.w) * COLS + c) * PART;
    const float* rest = p.part + (2 * (int64_t)(run + 1) * COLS + c) * PART;           // the next runs begin in this work
    top = PA_NOTHING;
    sum = 0.f;
    a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i0 = begin; i0 < item.z; i0 += stride * PM_DEPTH) {
      float2 ml[PM_DEPTH];
      float4 v[PM_DEPTH];
#pragma unroll
      for (int k = 0; k < PM_DEPTH; ++k) {
        const int i = i0 + k * stride;
        const float* rec = i == 0 ? first : rest + (int64_t)(i - 1) * 2 * COLS * PART;
        ml[k] = i < item.z ? *reinterpret_cast<const float2*>(rec) : make_float2(PA_NOTHING, 0.f);
        v[k] = i < item.z ? *reinterpret_cast<const float4*>(rec + 4 + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < PM_DEPTH; ++k) add(ml[k].x, ml[k].y, v[k]);
    }
  };
  auto put = [&](int4 item) {
    const PagedSeq seq = paged_seq(p.c, item.x - 1, p.rows);
    const int groups = paged_share<COLS>(p, seq).groups, kv = item.y / groups, cc = (item.y - kv * groups) * COLS + c;
    if (cc >= seq.n_new * p.ratio) return;
    const int tok = p.over_ratio(cc);
    const int64_t row = (int64_t)(seq.first + tok) * p.n_q + kv * p.ratio + cc - tok * p.ratio;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>((T*)p.out + row * HD + 4 * lane) = make_uint2(Pair<T>::put(a.x * inv, a.y * inv), Pair<T>::put(a.z * inv, a.w * inv));
    if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? neg_inf() : (top + log2f(sum)) * LN2;
  };
  if (items[w].x != 0 && items[w].z <= PM_DEPTH) {
    gather(run0 + w, items[w], 0, 1);
    put(items[w]);
  }
#pragma unroll 1
  for (int k = 0; k < PM_RUNS; ++k) {
    const int4 item = items[k];
    if (item.z <= PM_DEPTH) continue;
    gather(run0 + k, item, w, PM_RUNS);
    __syncthreads();
    float* mine = acc_s[w][c];
    if (lane == 0) *reinterpret_cast<float2*>(mine) = make_float2(top, sum);
    *reinterpret_cast<float4*>(mine + 4 + 4 * lane) = a;
    __syncthreads();
    if (w != 0) continue;
#pragma unroll
    for (int i = 1; i < PM_RUNS; ++i) {
      const float* rec = acc_s[i][c];
      add(rec[0], rec[1], *reinterpret_cast<const float4*>(rec + 4 + 4 * lane));
    }
    put(item);
  }
}

struct PagedAttnLayout {
  int grid, cols;
  bool tiles;                                            // a sequence may have more rows than are this kernel's
  size_t part, tile, bytes;
};
static PagedAttnLayout paged_attn_layout(int ratio, int max_new) {
  PagedAttnLayout l;
  l.grid = (sm_count() > 0 ? sm_count() : 1) * PA_CTAS;
  l.cols = (int64_t)ratio * max_new <= 4 ? 4 : 8;
  l.part = ((size_t)l.grid * sizeof(int4) + 127) & ~(size_t)127;
  l.tile = (l.part + (size_t)l.grid * (2 * l.cols * PART + PA_WARPS * PA_HELD) * 4 + 127) & ~(size_t)127;
  l.tiles = (int64_t)ratio * max_new > PA_SHORT_ROWS;
  l.bytes = l.tile + (l.tiles ? paged_tile_bytes() : 0);
  return l;
}

static constexpr size_t split_smem(int n_seqs) { return (size_t)PA_WARPS * PA_STAGES * PA_GROUP * PG_BYTES + (size_t)(n_seqs + 1) * 8; }

template <typename T, int COLS>
static cudaError_t launch_paged_split(const PagedAttnParams& p, int grid, cudaStream_t st) {
  // Asked for once on a device, for the most that a call can need: the limit belongs to the kernel, not to the call, and
  // another thread's call may be between its request and its launch.
  static std::atomic<bool> configured[MAX_DEVICES];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(paged_split_kernel<T, COLS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)split_smem(SHARD_PAGED_MAX_SEQS));
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(32 * PA_WARPS);
  cfg.dynamicSmemBytes = split_smem(p.c.n_seqs);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, paged_split_kernel<T, COLS>, p);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3((grid + PM_RUNS - 1) / PM_RUNS);
  cfg.blockDim = dim3(32 * COLS * PM_RUNS);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_merge_kernel<T, COLS>, p, grid);
}

}  // namespace shard

using namespace shard;

extern "C" size_t shard_b200_paged_attn_workspace_bytes(const ShardPaged* cache_host, int32_t n_q, int32_t rows, int32_t max_new) {
  if (paged_check(cache_host, rows) != SHARD_OK || n_q < 1 || n_q > 65536 || n_q % cache_host->nkv || max_new < 0) return 0;
  return paged_attn_layout(n_q / cache_host->nkv, max_new).bytes;
}

extern "C" int shard_b200_paged_attn(const ShardPaged* cache_host, const void* q, int64_t q_tok_stride, int64_t q_head_stride, int32_t n_q,
                                     int32_t rows, int32_t max_new, int32_t dtype, float scale, void* out, float* lse, void* workspace,
                                     size_t workspace_bytes, int* status_dev, void* stream) {
  const int rc = paged_check(cache_host, rows);
  if (rc != SHARD_OK) return rc;
  if (!q || !out || !workspace || n_q < 1 || n_q > 65536 || n_q % cache_host->nkv || max_new < 0 || (dtype != SHARD_F16 && dtype != SHARD_BF16) ||
      !(scale == scale) || scale > 3e38f || scale < -3e38f)
    return SHARD_E_ARG;
  const PagedAttnLayout l = paged_attn_layout(n_q / cache_host->nkv, max_new);
  if (workspace_bytes < l.bytes) return SHARD_E_WORKSPACE;
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15) || ((uintptr_t)lse & 3) || ((q_tok_stride | q_head_stride) & 7))
    return SHARD_E_ALIGN;
  if (rows == 0 || cache_host->n_seqs == 0) return SHARD_OK;
  if ((int64_t)rows * n_q > INT32_MAX || (int64_t)cache_host->n_pages * cache_host->nkv * (cache_host->page_size / PG_BLOCK) >= UINT32_MAX)
    return SHARD_E_TOO_LARGE;
  PagedAttnParams p{*cache_host, q, q_tok_stride, q_head_stride, out, lse, status_dev, (float*)((unsigned char*)workspace + l.part),
                    (int4*)workspace, scale, n_q, rows, max_new, 0, PA_SHORT_ROWS, 0, 0, 0};
  p.set_ratio(n_q / cache_host->nkv);
  while ((PG_BLOCK << p.page_log2) < cache_host->page_size) ++p.page_log2;
  cudaStream_t st = (cudaStream_t)stream;
  // (rows that nobody has may be among them: then a sequence is short after all, and the tiles' kernel takes it)
  const bool all_long = l.tiles && (int64_t)p.c.n_seqs * max_new == rows;
  cudaError_t e = cudaSuccess;
  if (all_long) p.short_rows = 0;
  else
    e = dtype == SHARD_F16 ? (l.cols == 4 ? launch_paged_split<__half, 4>(p, l.grid, st) : launch_paged_split<__half, 8>(p, l.grid, st))
                           : (l.cols == 4 ? launch_paged_split<__nv_bfloat16, 4>(p, l.grid, st) : launch_paged_split<__nv_bfloat16, 8>(p, l.grid, st));
  if (e == cudaSuccess && l.tiles) e = launch_paged_tile(p, dtype == SHARD_BF16, (unsigned char*)workspace + l.tile, st);
  return e == cudaSuccess ? SHARD_OK : (int)e;
}
