// Attention over the paged 4-bit cache for sequences with many query rows to a KV head: a piece of a prompt, the next
// turn of a chat, drafted tokens.  Dense products on the tensor core, keys and values unpacked on the way.
//
// Units of work are 256 query rows of a sequence and KV head, in steps of two jobs; every CTA (one on each SM) takes
// an equal run of steps of all units, and partial results of units that several CTAs share are joined in order by
// paged_tile_merge_kernel.  Where there are fewer units than CTAs, each is cut into equal parts instead, about as long:
// a run over the end of one unit into the next would pay for a second start and a second result (5 us).  A job is
// S = Q K^T, softmax, O += P V for 128 rows and a tile of 128 keys:
//   - rows 0-127 belong to group A, 128-255 to group B; a step is one tile of keys, one job for each group;
//   - units of up to 128 rows have a step of two tiles instead: A takes the even ones, B the odd ones, for the same
//     rows.  Up to 64 (32) rows are there twice (four times), each copy for half (a quarter) of a tile's keys, so that
//     all warps have some.  At the end the shares of a row become one.
// While one group's products run, the other has the exponentials to itself.
//
//   warps 0-3, 4-7  groups A and B, thread = row: scores from tensor memory -> weights, written over them
//   warps 8-11      thread = token: 64 bytes of codes -> 128 fp16 numbers in the operand layout (exact), keys a tile
//                   ahead of values
//   warp 12         all products; 13: which values are no numbers (14 and 15 only give their registers away)
//
// The eight channels of a 32-bit word are unpacked in the order 0 4 1 5 2 6 3 7, in which two nibbles at a time leave
// it; queries are staged in that order, and the output is put back.  Weights are two fp16 parts (22 bits, as in
// paged_attn.cu), each product run twice: with the first part alone bf16 outputs would take two thirds of the time, and
// one in twenty would be a last place off.
//
// What bounds it: the chain of a step, 4 200 cycles a job: products with the weights, their end, scores, and the
// softmax of 128 numbers a thread, which the other group's products hide only in part and whose straight line of
// instructions is more than their cache holds (after tensor memory, the longest waits are for those).  2 048 rows x 4 query
// heads behind 8 192 tokens, 8 KV heads (309 GFLOP): 650 us, 475 TFLOP/s, bf16 and fp16 alike.  Start
// and result of a piece are some 8 000 cycles each.  Measured and slower: a thread for each group's products (470 us),
// eight unpacking warps with the scores read from tensor memory twice (485 us).
#include <atomic>

#include "paged_attn.cuh"

namespace shard {

constexpr int PT_UNPACK_WARP = 8, PT_MMA_WARP = 12;
constexpr int PT_THREADS = 32 * (PT_MMA_WARP + 4);       // (registers change hands by fours of warps)
// Registers of a thread, whose sum over the four fours of warps is what the block is launched with (128 each).  A row's
// 128 scores are to stay in registers: reading them from tensor memory a second time takes 200 cycles for every 32.
constexpr int PT_REGS_SOFTMAX = 200, PT_REGS_UNPACK = 80, PT_REGS_MMA = 32;
static_assert(2 * PT_REGS_SOFTMAX + PT_REGS_UNPACK + PT_REGS_MMA == 4 * 128, "no more than the block was launched with");
constexpr int PT_ROWS = 256;                             // of a unit
constexpr int PT_KEYS = 128;                             // of a tile
constexpr int PT_TILE_BYTES = 32768;
constexpr int PT_COL_O = 256;                            // score columns of A, B; accumulators of A, B
constexpr int PT_BARS = 19;
constexpr int PT_HOLD = 16;                              // tiles of a group whose products add up in the accumulator (see paged_attn.cuh)
constexpr int PT_TRIES = 3;                              // lengths of parts that are tried
constexpr int PT_WALK_BYTES = 128;
constexpr int PT_SMEM = 1024 + 6 * PT_TILE_BYTES + PT_BARS * 8 + 16 + 256 * 8 + 256 * 4 + 32 + (PT_THREADS + 1) * 8 + (PT_THREADS / 32) * PT_WALK_BYTES + 8;

// ---- the list of work ----------------------------------------------------------------------------
struct TileUnits {
  int cols, count;                                       // query rows of a KV head; units of 256 of them
  int n_new, pos0, room;
  __device__ __forceinline__ int keys(const PagedAttnParams& p, int r) const {   // tiles of keys that unit r's rows see (at least one)
    const int last = min(p.over_ratio(min(PT_ROWS * (r + 1), cols) - 1), n_new - 1);
    return max((min(max(pos0 + last + 1, 0), room) + PT_KEYS - 1) / PT_KEYS, 1);
  }
  __device__ __forceinline__ bool two(int r) const { return cols - PT_ROWS * r > PT_ROWS / 2; }
  __device__ __forceinline__ int steps(const PagedAttnParams& p, int r) const { const int k = keys(p, r); return two(r) ? k : (k + 1) / 2; }
  __device__ __forceinline__ int parts(const PagedAttnParams& p, int r, int most) const {
    return (int)(((uint32_t)steps(p, r) + (uint32_t)most - 1) / (uint32_t)most);
  }
  __device__ __forceinline__ int parts_of_head(const PagedAttnParams& p, int most) const {
    int s = 0;
    for (int r = 0; r < count; ++r) s += parts(p, r, most);
    return s;
  }
  __device__ __forceinline__ int64_t steps_of_head(const PagedAttnParams& p) const {
    int64_t s = 0;
    for (int r = 0; r < count; ++r) s += steps(p, r);
    return s;
  }
};
__device__ __forceinline__ TileUnits tile_units(const PagedAttnParams& p, const PagedSeq& s) {
  TileUnits u;
  u.n_new = s.n_new;
  u.pos0 = s.pos0;
  u.room = min(s.len, p.c.table_width * p.c.page_size);
  u.cols = s.n_new * p.ratio;
  u.count = s.n_new > p.max_new || u.cols <= p.short_rows ? 0 : (u.cols + PT_ROWS - 1) / PT_ROWS;
  return u;
}

// A CTA's run of the list, unit by unit.  Every warp walks it for itself, in shared memory: registers are scarce.
struct TileWalk {
  int parts;                                             // of the unit, where units are cut into parts; 0: runs
  int64_t left;                                          // steps of the run that are still to come
  int b, kv, r, step;                                    // where the next one is
  TileUnits u;
  // the piece that `next` has found
  int seq_first, k0, k1, all_keys;                       // tiles of keys k0 .. k1 - 1 of all_keys
  bool two, whole, opens;                                // opens: it begins with the unit's first step

  __device__ __forceinline__ void load(const PagedAttnParams& p) {
    const PagedSeq s = paged_seq(p.c, b, p.rows);
    seq_first = s.first;
    u = tile_units(p, s);
  }
  // `chunks`: steps before every chunk of `each` sequences
  __device__ __forceinline__ void init(const PagedAttnParams& p, const int64_t* chunks, int n_chunks, int each, int64_t begin, int64_t end) {
    parts = 0;
    left = end - begin;
    if (left <= 0) return;
    int lo = 0, hi = n_chunks;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (chunks[mid] <= begin) lo = mid; else hi = mid;
    }
    int64_t at = begin - chunks[lo];
    for (b = lo * each;; ++b) {
      load(p);
      if (u.count == 0) continue;
      const int64_t head = u.steps_of_head(p);
      if (at < head * p.c.nkv) {
        kv = (int)pa_div(at, head);
        at -= kv * head;
        break;
      }
      at -= head * p.c.nkv;
    }
    for (r = 0; at >= u.steps(p, r); ++r) at -= u.steps(p, r);
    step = (int)at;
  }
  // The CTA's part where units are cut into parts of at most `most` steps: a walk of one piece.  `chunks`: parts before.
  __device__ __forceinline__ void init_part(const PagedAttnParams& p, const int64_t* chunks, int n_chunks, int each, int most) {
    left = 0;
    if (blockIdx.x >= chunks[PT_THREADS]) return;
    int lo = 0, hi = n_chunks;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (chunks[mid] <= blockIdx.x) lo = mid; else hi = mid;
    }
    int at = (int)(blockIdx.x - chunks[lo]);
    for (b = lo * each;; ++b) {
      load(p);
      if (u.count == 0) continue;
      const int head = u.parts_of_head(p, most);
      if (at < head * p.c.nkv) {
        kv = (int)((uint32_t)at / (uint32_t)head);
        at -= kv * head;
        break;
      }
      at -= head * p.c.nkv;
    }
    for (r = 0; at >= u.parts(p, r, most); ++r) at -= u.parts(p, r, most);
    parts = u.parts(p, r, most);
    const uint32_t n = u.steps(p, r);                    // (2^23 at most, and fewer parts than CTAs)
    step = (int)(n * (uint32_t)at / (uint32_t)parts);
    left = (int)(n * (uint32_t)(at + 1) / (uint32_t)parts) - step;
  }
  __device__ __forceinline__ bool next(const PagedAttnParams& p) {
    if (left <= 0) return false;
    if (r == u.count) {                                  // the unit before was its head's last
      r = 0;
      if (++kv == p.c.nkv) {
        kv = 0;
        do { ++b; load(p); } while (u.count == 0);
      }
    }
    two = u.two(r);
    all_keys = u.keys(p, r);
    const int steps = two ? all_keys : (all_keys + 1) / 2, n = (int)min((int64_t)(steps - step), left);
    unit = r;
    opens = step == 0;
    whole = opens && n == steps;
    k0 = two ? step : 2 * step;
    k1 = two ? step + n : min(2 * (step + n), all_keys);
    left -= n;
    rest_steps = steps - step - n;
    step += n;
    if (step == steps) { step = 0; ++r; }
    return true;
  }
  int unit, rest_steps;                                  // its number among the head's units; the unit's steps behind the piece
};
static_assert(sizeof(TileWalk) <= PT_WALK_BYTES, "a walk has its place");

// ---- unpacking -----------------------------------------------------------------------------------
// A token's vector, a thread's work: 16 words -> 16 pieces of 8 fp16 numbers in row `row` of a 128-byte-swizzled tile.
__device__ __forceinline__ void tile_unpack(unsigned char* tile, int row, const uint4 (&raw)[4], uint32_t par, uint32_t magic) {
  const __half2 k16 = __float2half2_rn(16.f), kb = __float2half2_rn(-15360.f), k1_16 = __float2half2_rn(0.0625f);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t one = h ? __byte_perm(par, par, 0x3232) : __byte_perm(par, par, 0x1010);
    const __half2 s = as_half2(one & 0xfff0fff0u), s16 = __hmul2(s, k1_16);
    const __half2 z = as_half2(pa_1024(one, 0x000f000fu, magic)), z16 = __hfma2(z, k16, kb);
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const uint4 q = raw[g >> 1];
      const uint32_t w = (g & 1) ? (h ? q.w : q.z) : (h ? q.y : q.x), w8 = w >> 8;
      uint4 o;
      o.x = as_u32(__hmul2(__hsub2(as_half2(pa_1024(w, 0x000f000fu, magic)), z), s));
      o.y = as_u32(__hmul2(__hsub2(as_half2(pa_1024(w, 0x00f000f0u, magic)), z16), s16));
      o.z = as_u32(__hmul2(__hsub2(as_half2(pa_1024(w8, 0x000f000fu, magic)), z), s));
      o.w = as_u32(__hmul2(__hsub2(as_half2(pa_1024(w8, 0x00f000f0u, magic)), z16), s16));
      *reinterpret_cast<uint4*>(tile + h * 16384 + sw128_off(row, g)) = o;
    }
  }
}

// A bounded wait as mbar_wait is (tens of milliseconds at least), without a time to sleep: with one, the warps that wait
// issue three quarters of all instructions, most of them between two naps.
// (HEED: someone else giving up ends it too)
constexpr int PT_WAIT_TRIES = 1 << 20;
template <bool HEED = true>
__device__ __forceinline__ bool tile_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (int i = 0; i < PT_WAIT_TRIES; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if (HEED && (i & 63) == 63 && *abort_flag) break;
  }
  *abort_flag = 1;
  return false;
}
// The same for what may take as long as a whole piece of work does: the bound counts from the last time that `progress`,
// which whoever is waited for moves on with every tile, was seen to change.  There is time to sleep here.
constexpr int PT_LONG_TRIES = 1 << 15;                   // of some 2 microseconds
__device__ __forceinline__ bool long_wait(uint32_t bar, uint32_t parity, const volatile int* progress, volatile int* abort_flag) {
  int seen = *progress;
  for (int i = 0; i < PT_LONG_TRIES; ++i) {
    if (mbar_try(bar, parity, 1000)) return true;
    if (*abort_flag) return false;
    const int now = *progress;
    if (now != seen) i = 0;
    seen = now;
    __nanosleep(1000);
  }
  *abort_flag = 1;
  return false;
}
// two fp32 operations in an instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
// single-thread forms of the products (the caller is one thread)
__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <int N>
__device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// ---- the kernel ----------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(PT_THREADS, 1) paged_tile_kernel(const __grid_constant__ PagedAttnParams p) {
  extern __shared__ __align__(128) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* q_s = smem;                             // [group]
  unsigned char* k_s = q_s + 2 * PT_TILE_BYTES;          // [stage]
  unsigned char* v_s = k_s + 2 * PT_TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + 2 * PT_TILE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + PT_BARS);
  volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* ml_s = reinterpret_cast<float2*>(tmem_slot + 4);         // reference points and sums of rows that several threads have
  float* f_s = reinterpret_cast<float*>(ml_s + 256);               // of a row
  int* tally = reinterpret_cast<int*>(f_s + 256);
  volatile int* jobs_done = tally + PT_TRIES + 1;                  // moves on with the products,
  volatile int* looked_at = tally + PT_TRIES + 2;                  // and with the tiles whose values have been looked through
  int64_t* chunks = reinterpret_cast<int64_t*>(tally + 8);        // [threads + 1] steps before each thread's sequences
  int2* odd_s = reinterpret_cast<int2*>(reinterpret_cast<unsigned char*>(chunks + PT_THREADS + 1) + (PT_THREADS / 32) * PT_WALK_BYTES);   // first token of the piece whose values (of each half) are no numbers
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  auto K_FULL = [&](int s) { return bar(s); };           // keys unpacked
  auto K_FREE = [&](int s) { return bar(2 + s); };       // their last product has run
  auto V_FULL = [&](int s) { return bar(4 + s); };
  auto V_FREE = [&](int s) { return bar(6 + s); };
  auto S_FULL = [&](int g) { return bar(8 + g); };       // scores complete
  auto P_READY = [&](int g) { return bar(10 + g); };     // weights written, accumulator rescaled
  auto O_DONE = [&](int g) { return bar(12 + g); };      // the product with the weights has run
  const uint32_t Q_READY = bar(14), X_FULL = bar(15), X_FREE = bar(16), DRAINED = bar(17), ODD_READY = bar(18);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_launch();
  griddep_wait();

  const int n_seqs = p.c.n_seqs, each = (n_seqs + PT_THREADS - 1) / PT_THREADS, n_chunks = (n_seqs + each - 1) / each;
  if (tid < 8) tally[tid] = 0;
  __syncthreads();
  {
    int64_t sum = 0;
    int units = 0;
    for (int b = tid * each; b < min((tid + 1) * each, n_seqs); ++b) {
      const PagedSeq s = paged_seq(p.c, b, p.rows);
      const TileUnits u = tile_units(p, s);
      if (p.short_rows == 0 && blockIdx.x == 0 && p.status && s.n_new > 0) {   // (otherwise the other kernel has looked)
        if (s.n_new > p.max_new) atomicOr(p.status, PG_BAD_COUNT);
        else if (s.len > u.room) atomicOr(p.status, PG_BAD_PAGE);
      }
      sum += u.steps_of_head(p) * p.c.nkv;
      units = min(units + u.count * p.c.nkv, 1 << 20);
    }
    chunks[tid] = sum;
    if (units > 0) atomicAdd(&tally[PT_TRIES], units);
  }
  if (warp == PT_MMA_WARP) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(K_FULL(i), 4); mbar_init(K_FREE(i), 1); mbar_init(V_FULL(i), 4); mbar_init(V_FREE(i), 1);
        mbar_init(S_FULL(i), 1); mbar_init(P_READY(i), 4); mbar_init(O_DONE(i), 1);
      }
      mbar_init(Q_READY, 8); mbar_init(X_FULL, 8); mbar_init(X_FREE, 8); mbar_init(DRAINED, 1); mbar_init(ODD_READY, 1);
      *abort_s = 0;
      fence_mbar_init();
    }
  }
  __syncthreads();
  auto add_up = [&]() {                                  // exclusive sums of what the threads have in `chunks`
    if (warp != 0) return;
    int64_t carry = 0;
    for (int i0 = 0; i0 < n_chunks; i0 += 32) {
      const int64_t mine = chunks[i0 + lane];
      int64_t incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      chunks[i0 + lane] = carry + incl - mine;
      carry += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) chunks[PT_THREADS] = carry;
  };
  add_up();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int64_t total = chunks[PT_THREADS], n_ctas = min((int64_t)gridDim.x, total);
  // runs of `per` steps, the first `more` of them one longer
  const int64_t per = n_ctas > 0 ? pa_div(total, n_ctas) : 0, more = total - per * n_ctas;
  const bool works = blockIdx.x < n_ctas;
  const int64_t begin = works ? per * blockIdx.x + min((int64_t)blockIdx.x, more) : 0, end = works ? begin + per + (blockIdx.x < more) : 0;
  if (tid == 0) p.items[blockIdx.x] = make_int4(0, 0, 0, 0);
  TileWalk& walk = *reinterpret_cast<TileWalk*>(reinterpret_cast<unsigned char*>(chunks + PT_THREADS + 1) + warp * PT_WALK_BYTES);
  int most = 0;                                          // longest part; 0: runs
  if (total > 0 && tally[PT_TRIES] <= (int)gridDim.x) {
    // a little longer parts than the runs would be, as far as there are CTAs for them
    int longest[PT_TRIES], count[PT_TRIES] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < PT_TRIES; ++i) longest[i] = (int)min(per + 1 + ((per + 1) << i) / 8, (int64_t)1 << 30);   // an eighth, a quarter, half more
    for (int b = tid * each; b < min((tid + 1) * each, n_seqs); ++b) {
      const TileUnits u = tile_units(p, paged_seq(p.c, b, p.rows));
#pragma unroll
      for (int i = 0; i < PT_TRIES; ++i)
        if (u.count > 0) count[i] += u.parts_of_head(p, longest[i]) * p.c.nkv;
    }
#pragma unroll
    for (int i = 0; i < PT_TRIES; ++i)
      if (count[i] > 0) atomicAdd(&tally[i], count[i]);
    __syncthreads();
#pragma unroll
    for (int i = PT_TRIES - 1; i >= 0; --i)
      if (tally[i] <= (int)gridDim.x) most = longest[i];
    if (most > 0) {
      int64_t sum = 0;
      for (int b = tid * each; b < min((tid + 1) * each, n_seqs); ++b) {
        const TileUnits u = tile_units(p, paged_seq(p.c, b, p.rows));
        if (u.count > 0) sum += (int64_t)u.parts_of_head(p, most) * p.c.nkv;
      }
      chunks[tid] = sum;
      __syncthreads();
      add_up();
      __syncthreads();
    }
  }
  if (lane == 0) {
    if (most > 0) walk.init_part(p, chunks, n_chunks, each, most);
    else walk.init(p, chunks, n_chunks, each, begin, end);
  }
  auto next_piece = [&]() {                              // (a whole warp)
    bool found = false;
    __syncwarp();                                        // all lanes are done with the piece before
    if (lane == 0) found = walk.next(p);
    __syncwarp();
    return __shfl_sync(0xffffffffu, (int)found, 0) != 0;
  };

  if (warp >= PT_MMA_WARP) {
    fewer_regs<PT_REGS_MMA>();
    if (warp == PT_MMA_WARP && lane == 0) {
      // One thread, the groups in turn: while it waits for one group's product, the other has the exponentials to itself.
      // (A thread for each group let them fall into step, both at the exponentials and then both at the products: 7 000
      // cycles a step.)
      constexpr uint32_t IDESC_S = umma_idesc(128, 128, false, false), IDESC_O = umma_idesc(128, 128, false, true);
      uint32_t tile0 = 0, jobs_a = 0, jobs_b = 0, pieces = 0;   // tiles of keys and jobs of each group before this piece
      bool ok = true;
      for (; ok && walk.next(p); ++pieces) {
        const bool two = walk.two;
        const int n_tiles = walk.k1 - walk.k0, n_jobs = two ? 2 * n_tiles : n_tiles, shift = two ? 1 : 0;
        ok = tile_wait(Q_READY, pieces & 1, abort_s);
        if (!ok) break;
        tc_fence_after();
        const uint32_t q_at = smem_u32(q_s), k_at = smem_u32(k_s), v_at = smem_u32(v_s);
        auto scores = [&](int j) {
          const int g = j & 1;
          const uint32_t t = tile0 + (uint32_t)(j >> shift), st = t & 1;
          if (!tile_wait(K_FULL(st), (t >> 1) & 1, abort_s)) return false;
          tc_fence_after();
          const uint64_t qd = smem_desc_sw128(q_at + (two ? g * PT_TILE_BYTES : 0), 16, 1024);
          const uint64_t kd = smem_desc_sw128(k_at + st * PT_TILE_BYTES, 16, 1024);
          const uint32_t S = tmem + 128 * g;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint64_t adv = (uint64_t)(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4);
            product_ss(S, qd + adv, kd + adv, IDESC_S, ks > 0 ? 1u : 0u);
          }
          commit(S_FULL(g));
          if (!two || g == 1) commit(K_FREE(st));
          return true;
        };
#pragma unroll 1
        for (int j = -2; j < n_jobs && ok; ++j) {        // (the first two turns only begin the groups' first scores)
          const int g = j & 1;
          if (j >= 0) {
            const uint32_t t = tile0 + (uint32_t)(j >> shift), st = t & 1, job = (g ? jobs_b : jobs_a) + (uint32_t)(j >> 1);   // (no array: this thread waits for nothing in memory)
            ok = tile_wait(V_FULL(st), (t >> 1) & 1, abort_s) && tile_wait(P_READY(g), job & 1, abort_s);
            if (!ok) break;
            tc_fence_after();
            const uint64_t vd = smem_desc_sw128(v_at + st * PT_TILE_BYTES, 16384, 1024);
            const uint32_t S = tmem + 128 * g, O = tmem + PT_COL_O + 128 * g;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {             // weights of 32 tokens lie in 32 columns, first parts in front
              const uint32_t w = S + 32 * (ks >> 1) + 8 * (ks & 1);
              product_ts(O, w, vd + (uint64_t)((ks * 2048) >> 4), IDESC_O, ((j >> 1) % PT_HOLD != 0 || ks > 0) ? 1u : 0u);
              product_ts(O, w + 16, vd + (uint64_t)((ks * 2048) >> 4), IDESC_O, 1u);
            }
            commit(O_DONE(g));
            *jobs_done = (int)(2 * tile0) + j;
            if (!two || g == 1) commit(V_FREE(st));
            // the next scores take the place of the weights
            if (j + 2 < n_jobs) ok = tile_wait(O_DONE(g), job & 1, abort_s);
          }
          if (ok && j + 2 < n_jobs) ok = scores(j + 2);
        }
        tile0 += (uint32_t)n_tiles;
        jobs_a += (uint32_t)(n_jobs + 1) / 2;
        jobs_b += (uint32_t)n_jobs / 2;
      }
      // whoever gave up: do not leave before the tensor core is done with this CTA's memory (for as long as a product can take)
      commit(DRAINED);
      tile_wait<false>(DRAINED, 0, abort_s);
    } else if (warp == PT_MMA_WARP + 1) {
      // Values that are no numbers, which the unpacking warps leave out: the first token of each half.
      for (uint32_t pieces = 0; next_piece(); ++pieces) {
        const int32_t* table = p.c.page_table + walk.b * p.c.table_stride;
        const int room = walk.u.room, k1 = walk.k1;
        constexpr int AHEAD = 2;                         // tiles in flight; a lane has four tokens' words of each
        int first0 = INT_MAX, first1 = INT_MAX;
#pragma unroll 1
        for (int tile = walk.k0; tile < k1; tile += AHEAD) {
          uint4 w[AHEAD];
          int at[AHEAD];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            const int blk = (tile + i) * (PT_KEYS / PG_BLOCK) + (lane >> 2);
            at[i] = blk * PG_BLOCK + 2 * (lane & 3);
            const int page = tile + i < k1 && blk * PG_BLOCK < room ? table[blk >> p.page_log2] : -1;
            w[i] = make_uint4(0u, 0u, 0u, 0u);
            if ((unsigned)page < (unsigned)p.c.n_pages)
              w[i] = *reinterpret_cast<const uint4*>(p.c.pool + (((int64_t)page * p.c.nkv + walk.kv) * (p.c.page_size / PG_BLOCK) + (blk & ((1 << p.page_log2) - 1))) * PG_BYTES +
                                                     PG_VP + 16 * (lane & 3));
          }
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {              // (what lies behind the last token is seen by nobody)
            first0 = min(first0, first_bad(bad_words(w[i].x), bad_words(w[i].y), at[i]));
            first1 = min(first1, first_bad(bad_words(w[i].z), bad_words(w[i].w), at[i]));
          }
          if (lane == 0) *looked_at = tile;
        }
        first0 = (int)__reduce_min_sync(0xffffffffu, (uint32_t)first0);
        first1 = (int)__reduce_min_sync(0xffffffffu, (uint32_t)first1);
        // (everyone is done with the piece before: this warp may be as far ahead as a whole piece)
        const bool gave_up = !long_wait(Q_READY, pieces & 1, jobs_done, abort_s);
        if (__any_sync(0xffffffffu, gave_up)) break;
        if (lane == 0) {
          *odd_s = make_int2(first0, first1);
          mbar_arrive(ODD_READY);
        }
      }
    }
    __syncwarp();
  } else if (warp >= PT_UNPACK_WARP) {
    // ---- unpacking: thread = token of the tile
    fewer_regs<PT_REGS_UNPACK>();
    const int tok = tid & 127, in_block = tok & (PG_BLOCK - 1);
    uint32_t magic;
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
    const int64_t per_head = (int64_t)(p.c.page_size / PG_BLOCK) * PG_BYTES;
    // the tiles of all pieces, one behind the other: the page is looked up two tiles ahead, the bytes loaded one
    int tile = 0, last = 0, room = 0, kv = 0;
    const int32_t* table = nullptr;
    auto advance = [&]() {                               // the next tile; false behind the last
      if (tile < last) { ++tile; return true; }
      if (!next_piece()) return false;
      tile = walk.k0;
      last = walk.k1 - 1;
      room = walk.u.room;
      kv = walk.kv;
      table = p.c.page_table + walk.b * p.c.table_stride;
      return true;
    };
    struct Place { int page, blk, kv; bool there; };
    auto look_up = [&]() {
      const int blk = tile * (PT_KEYS / PG_BLOCK) + (tok >> 4);
      Place x{-1, blk, kv, blk * PG_BLOCK + in_block < room};
      if (x.there) x.page = table[blk >> p.page_log2];
      return x;
    };
    uint4 raw_k[4], raw_v[4];
    uint32_t par_k = 0, par_v0 = 0, par_v1 = 0;          // parameters: of keys both halves, of values each half
    auto block_of = [&](const Place& x) {
      return p.c.pool + ((int64_t)x.page * p.c.nkv + x.kv) * per_head + (x.blk & ((1 << p.page_log2) - 1)) * PG_BYTES;
    };
    // (no token, no page: zeros, which the scores leave out)
    auto load_keys = [&](const Place& x) {
      const bool good = (unsigned)x.page < (unsigned)p.c.n_pages;
      if (x.there && !good && in_block == 0 && p.status) atomicOr(p.status, PG_BAD_PAGE);
      par_k = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw_k[i] = make_uint4(0u, 0u, 0u, 0u);
      if (good) {
        const unsigned char* block = block_of(x);
#pragma unroll
        for (int i = 0; i < 4; ++i) raw_k[i] = reinterpret_cast<const uint4*>(block + in_block * 64)[i];
        par_k = *reinterpret_cast<const uint32_t*>(block + PG_KP + in_block * 4);
      }
    };
    auto load_values = [&](const Place& x) {
      par_v0 = par_v1 = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) raw_v[i] = make_uint4(0u, 0u, 0u, 0u);
      if ((unsigned)x.page < (unsigned)p.c.n_pages) {
        const unsigned char* block = block_of(x);
#pragma unroll
        for (int i = 0; i < 4; ++i) raw_v[i] = reinterpret_cast<const uint4*>(block + PG_V + in_block * 64)[i];
        par_v0 = *reinterpret_cast<const unsigned short*>(block + pg_vparam(in_block));
        par_v1 = *reinterpret_cast<const unsigned short*>(block + pg_vparam(in_block) + 8);
      }
    };
    auto hand_over = [&](uint32_t t, unsigned char* tiles, const uint4 (&raw)[4], uint32_t par, uint32_t bar_free, uint32_t bar_full, bool values) {
      const bool gave_up = t >= 2 && !tile_wait(bar_free, ((t >> 1) - 1) & 1, abort_s);
      if (__any_sync(0xffffffffu, gave_up)) return false;
      if (values) par &= ~bad_words(par);                // (0 * NaN is not 0: who sees them has them set at the end of the piece)
      tile_unpack(tiles + (t & 1) * PT_TILE_BYTES, tok, raw, par, magic);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_full);
      return true;
    };
    // Keys are a tile ahead of values: a stage of values is only free when both groups' softmax is done, and the next
    // scores should not wait for that.
    Place here{}, next{};
    bool has_next = advance();
    if (has_next) {
      next = look_up();
      load_keys(next);
    }
    bool has_here = false, has_values = false;
#pragma unroll 1
    for (uint32_t t = 0;; ++t) {                         // keys of tile t, values of tile t - 1
      has_here = has_next;
      here = next;
      has_next = has_here && advance();
      if (has_next) next = look_up();
      if (has_here && !hand_over(t, k_s, raw_k, par_k, K_FREE(t & 1), K_FULL(t & 1), false)) break;
      if (has_next) load_keys(next);
      if (has_values && !hand_over(t - 1, v_s, raw_v, par_v0 | (par_v1 << 16), V_FREE((t - 1) & 1), V_FULL((t - 1) & 1), true)) break;
      if (!has_here) break;
      load_values(here);
      has_values = true;
    }
  } else {
    // ---- softmax: thread = row of the group
    more_regs<PT_REGS_SOFTMAX>();
    const int g = warp >> 2, row = tid & 127;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16, S = tmem + 128 * g + lane_off, O = tmem + PT_COL_O + 128 * g + lane_off;
    uint32_t job = 0, pieces = 0, frees = 0, fulls = 0;   // (uses of the barriers so far)
    bool bad = false;
    auto wait_for = [&](uint32_t which, uint32_t parity) {   // (a whole warp)
      const bool gave_up = !tile_wait(which, parity, abort_s);
      bad = __any_sync(0xffffffffu, gave_up);
      return !bad;
    };
    for (bool first_piece = true; !bad && next_piece(); first_piece = false) {
      const bool two = walk.two;
      const int k1 = walk.k1, room = walk.u.room;
      // units of few rows: copies of them in all four warps, each for its share of a tile's keys
      const int rows = min(walk.u.cols - walk.unit * PT_ROWS, PT_ROWS), copies = two || rows > 64 ? 1 : rows > 32 ? 2 : 4;
      const int copy_rows = 128 / copies, copy = row / copy_rows, r = two ? 128 * g + row : row % copy_rows;   // r: row of the unit
      const bool warp_live = (r & ~31) < rows;
      const int tok = p.over_ratio(walk.unit * PT_ROWS + r);
      // tokens that the row sees (rows that are none hide nothing)
      const int vis = r < rows ? min(max(walk.u.pos0 + tok + 1, 0), room) : room;
      // The queries, a row to 16 lanes: scaled by a power of two (largest channel 2^9 .. 2^10) and with the sign of
      // `scale`, in as many copies as there are.
      {
        const int c = lane & 15;
        const float mag = fabsf(p.scale) * LOG2E;
        const int from = two ? 128 * g + 32 * (warp & 3) : 4 * warp, n_log2 = two ? 5 : 2, skip = two ? 0 : 28;   // (one unit: four rows to a warp, then the next 32)
        constexpr int AHEAD = 2;
#pragma unroll 1
        for (int i0 = 0; i0 < (two ? 16 : copy_rows / 16); i0 += AHEAD) {
          uint4 u[AHEAD];
          int at[AHEAD];
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            const int k = 2 * (i0 + i) + (lane >> 4);
            at[i] = from + k + (k >> n_log2) * skip;
            const int cc = walk.unit * PT_ROWS + at[i], of_tok = p.over_ratio(cc);
            u[i] = make_uint4(0u, 0u, 0u, 0u);
            if (at[i] < rows)
              u[i] = reinterpret_cast<const uint4*>((const T*)p.q + (int64_t)(walk.seq_first + of_tok) * p.q_tok +
                                                    (walk.kv * p.ratio + cc - of_tok * p.ratio) * p.q_head)[c];
          }
#pragma unroll
          for (int i = 0; i < AHEAD; ++i) {
            const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
            float x[8], top = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 v = Pair<T>::get(w[e]);
              x[2 * e] = v.x;
              x[2 * e + 1] = v.y;
              top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const int ex = (int)(__float_as_uint(top) >> 23), up = top == 0.f || ex == 255 ? 127 : min(263 - ex, 250);
            const float back = __uint_as_float((uint32_t)(254 - up) << 23);
            const float by = p.scale == 0.f ? 0.f : copysignf(__uint_as_float((uint32_t)up << 23), p.scale);
            if (c == 0) f_s[at[i]] = p.scale == 0.f ? 1.f : fminf(fmaxf(back * mag, 1e-37f), PA_MOST_F);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= by;
            const uint4 v = make_uint4(pack_half2(x[0], x[4]), pack_half2(x[1], x[5]), pack_half2(x[2], x[6]), pack_half2(x[3], x[7]));
            unsigned char* tile = q_s + (two ? g * PT_TILE_BYTES : 0) + (c >> 3) * 16384;
            if (at[i] < copy_rows * (two ? 2 : 1))
              for (int k = 0; k < copies; ++k) *reinterpret_cast<uint4*>(tile + sw128_off((at[i] & 127) + k * copy_rows, c & 7)) = v;
          }
        }
      }
      fence_proxy_async();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(Q_READY);
      if (!wait_for(Q_READY, pieces++ & 1)) break;
      float f = f_s[r];                                  // what a score is times for the exponent of 2

      float ref = 0.f, lim = PA_NOTHING, l = 0.f;
      const int32_t* table = p.c.page_table + walk.b * p.c.table_stride;
      auto page_missing = [&](int tile) {                // lanes 0-7: whether the tile's block has no page
        const int blk = tile * (PT_KEYS / PG_BLOCK) + lane;
        return lane < PT_KEYS / PG_BLOCK && blk * PG_BLOCK < room && (unsigned)table[blk >> p.page_log2] >= (unsigned)p.c.n_pages;
      };
      const int stride = two ? 1 : 2, t_first = walk.k0 + (two ? 0 : g);
      bool missing = t_first < k1 && page_missing(t_first);
      bool fresh = true;                                 // no product in the accumulator yet
      // (a run has at most two pieces of units that others share: its first piece, and its last)
      auto records = [&]() { return p.part + (2 * (int64_t)blockIdx.x + (first_piece ? 0 : 1)) * PT_ROWS * PART; };
      // What the accumulator had before its last PT_HOLD tiles waits where the piece's result will go, four channels of
      // all lanes side by side: held = held * by + accumulator * scale.
      auto held = [&]() { return reinterpret_cast<float4*>(records() + (warp * 32) * PART) + lane; };
      auto held_by = [&]() {                             // (its reference point is behind it)
        float m;
        const float scale = pa_record(ref, f, f_s[r], m);
        return ex2(held()[32 * 32].x - m) / scale;
      };
      auto add_held = [&](uint32_t (&o)[16], int c, float scale, float by, bool has) {   // channels 16 c ..
        float4 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = has ? held()[(4 * c + i) * 32] : make_float4(0.f, 0.f, 0.f, 0.f);
        tmem_ld_x16(O + 16 * c, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) o[4 * i + e] = __float_as_uint(fmaf(x[e], by, __uint_as_float(o[4 * i + e]) * scale));
        }
      };
      for (int tile = t_first; tile < k1; tile += stride, ++job) {
        const uint32_t holes = __ballot_sync(0xffffffffu, missing);
        if (tile + stride < k1) missing = page_missing(tile + stride);
        if (!wait_for(S_FULL(g), job & 1)) break;
        tc_fence_after();
        if (!warp_live) {                                // (what its rows' weights are does not matter to the others')
          fresh = false;
          if (lane == 0) mbar_arrive(P_READY(g));
          continue;
        }
        const int limit = vis - PT_KEYS * tile;
        const bool edge = __any_sync(0xffffffffu, limit < PT_KEYS) || holes;
        float mx[4] = {neg_inf(), neg_inf(), neg_inf(), neg_inf()}, alpha = 1.f;
        float2 sum = make_float2(0.f, 0.f);
        const int c0 = copy * (4 / copies), c1 = c0 + 4 / copies;     // its quarters of the tile's keys
        if (copies > 1) {                                // no weights for the other copies' keys
          uint32_t zero[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) zero[i] = 0u;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            if (c >= c0 && c < c1) continue;
            tmem_st_x16(S + 32 * c, zero);
            tmem_st_x16(S + 32 * c + 16, zero);
          }
        }
        auto hide = [&](uint32_t (&s)[32], int c) {      // -infinity for what the row does not see of scores 32 c ..
          const int left = limit - 32 * c;
          uint32_t seen = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
          if ((holes >> (2 * c)) & 1) seen &= 0xffff0000u;
          if ((holes >> (2 * c)) & 2) seen &= 0x0000ffffu;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((seen >> i) & 1)) s[i] = 0xff800000u;
        };
        auto refer = [&]() {                             // the reference point follows
          const float most = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          if (fmaf(most, f, -ref) > lim) {
            alpha = pa_move(most, f_s[r], f, ref);
            if (lim != PA_MOST_LOG2) alpha = 0.f;
            lim = PA_MOST_LOG2;
          }
        };
        auto weigh = [&](const uint32_t (&s)[32], int c) {   // weights in the place of the scores
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 x = fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), make_float2(f, f), make_float2(-ref, -ref));
            const float2 w = make_float2(ex2(x.x), ex2(x.y));
            sum = add2(sum, w);
            hi[i] = pack_half2(w.x, w.y);
            const float2 rest = fma2(__half22float2(as_half2(hi[i])), make_float2(-1.f, -1.f), w);
            lo[i] = pack_half2(rest.x, rest.y);
          }
          tmem_st_x16(S + 32 * c, hi);
          tmem_st_x16(S + 32 * c + 16, lo);
        };
        if (copies == 1) {
          uint32_t s[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_x32(S + 32 * c, s[c]);
          tmem_wait_ld();
          if (edge) {
#pragma unroll
            for (int c = 0; c < 4; ++c) hide(s[c], c);
          }
#pragma unroll
          for (int i = 0; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i >> 5][i & 31]));
          refer();
#pragma unroll
          for (int c = 0; c < 4; ++c) weigh(s[c], c);
        } else {
          uint32_t s[32];
#pragma unroll 1
          for (int c = c0; c < c1; ++c) {
            tmem_ld_x32(S + 32 * c, s);
            tmem_wait_ld();
            if (edge) {
              hide(s, c);
              if (c != c1 - 1) {                         // (for the second pass)
                tmem_st_x16(S + 32 * c, *reinterpret_cast<uint32_t(*)[16]>(&s[0]));
                tmem_st_x16(S + 32 * c + 16, *reinterpret_cast<uint32_t(*)[16]>(&s[16]));
                tmem_wait_st();
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i]));
          }
          refer();
#pragma unroll 1
          for (int c = c1 - 1; c >= c0; --c) {           // (the last of its scores are still here)
            if (c != c1 - 1) {
              tmem_ld_x32(S + 32 * c, s);
              tmem_wait_ld();
            }
            weigh(s, c);
          }
        }
        l = l * alpha + (sum.x + sum.y);
        // (the group's product before this one has run: the scores were issued behind it)
        const int nth = (tile - t_first) >> (two ? 0 : 1);   // of the group's tiles of the piece
        if (nth % PT_HOLD == 0 && nth > 0) {             // the product to come begins the accumulator anew
          float m;
          const float scale = pa_record(ref, f, f_s[r], m), by = nth > PT_HOLD ? ex2(held()[32 * 32].x - m) : 0.f;
#pragma unroll 4
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16];
            add_held(o, c, alpha * scale, by, nth > PT_HOLD);
#pragma unroll
            for (int i = 0; i < 4; ++i) held()[(4 * c + i) * 32] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                                                            __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
          }
          held()[32 * 32] = make_float4(lim == PA_MOST_LOG2 ? m : PA_NOTHING, 0.f, 0.f, 0.f);
        } else if (!fresh && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t o[16];
            tmem_ld_x16(O + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_x16(O + 16 * c, o);
          }
        }
        fresh = false;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(P_READY(g));
      }
      if (bad || (!fresh && !wait_for(O_DONE(g), (job - 1) & 1))) break;
      tc_fence_after();

      // ---- the piece's result
      const bool finish = walk.whole;
      if (k1 - t_first > PT_HOLD * stride && warp_live) {                  // (the records that may lie there are written once all warps have read)
        const float by = held_by();
#pragma unroll 4
        for (int c = 0; c < 8; ++c) {
          uint32_t o[16];
          add_held(o, c, 1.f, by, true);
          tmem_st_x16(O + 16 * c, o);
        }
        tmem_wait_st();
        __syncwarp();
      }
      if (tid == 0 && walk.opens && !finish) {
        int pieces = walk.parts;
        if (pieces == 0) {
          const int64_t stop = end - walk.left + walk.rest_steps - 1;    // the unit's last step, and whose run that is in
          pieces = (int)(stop < (per + 1) * more ? pa_div(stop, per + 1) : more + pa_div(stop - (per + 1) * more, per)) - (int)blockIdx.x + 1;
        }
        p.items[blockIdx.x] = make_int4(walk.b + 1, walk.kv * walk.u.count + walk.unit, pieces, first_piece ? 0 : 1);
      }
      // a row of the unit: where its result goes
      auto row_of = [&](int of_unit) {
        const int cc = walk.unit * PT_ROWS + of_unit;
        const int tok = p.over_ratio(cc);
        return finish ? (int64_t)(walk.seq_first + tok) * p.n_q + walk.kv * p.ratio + cc - tok * p.ratio : (int64_t)of_unit;
      };
      auto put_sums = [&](int64_t at, float m, float sum) {
        if (!finish) *reinterpret_cast<float2*>(records() + at * PART) = make_float2(m, sum);
        else if (p.lse) p.lse[at] = sum == 0.f ? neg_inf() : (m + log2f(sum)) * LN2;
      };
      // eight channels from 8 c on of a row; the products leave them in the order 0 4 1 5 2 6 3 7
      auto put8 = [&](int64_t at, int c, const float (&x)[8]) {
        if (!finish) {
          float4* dst = reinterpret_cast<float4*>(records() + at * PART + 4 + 8 * c);
          dst[0] = make_float4(x[0], x[2], x[4], x[6]);
          dst[1] = make_float4(x[1], x[3], x[5], x[7]);
        } else {
          *reinterpret_cast<uint4*>((T*)p.out + at * HD + 8 * c) =
              make_uint4(Pair<T>::put(x[0], x[2]), Pair<T>::put(x[4], x[6]), Pair<T>::put(x[1], x[3]), Pair<T>::put(x[5], x[7]));
        }
      };
      float m;
      const float scale = pa_record(ref, f, f_s[r], m);
      if (lim != PA_MOST_LOG2) m = PA_NOTHING;
      l *= scale;
      {
        const bool gave_up = !long_wait(ODD_READY, (pieces - 1) & 1, looked_at, abort_s);
        bad = __any_sync(0xffffffffu, gave_up);
        if (bad) break;
      }
      const int odd_0 = odd_s->x, odd_1 = odd_s->y;
      if (two) {
        const bool live = r < rows;
        const float inv = !finish ? scale : l == 0.f ? 0.f : scale / l;
        const int64_t at = row_of(r);
        if (live) put_sums(at, m, l);
#pragma unroll 1
        for (int c = 0; c < 16 && warp_live; ++c) {
          uint32_t o[8];
          float x[8];
          tmem_ld_x8(O + 8 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = (c < 8 ? odd_0 : odd_1) < vis ? __uint_as_float(0x7fffffffu) : __uint_as_float(o[i]) * inv;
          if (live) put8(at, c, x);
          __syncwarp();
        }
      } else {
        // Groups and copies have a share of every row each.  They meet in shared memory, 64 channels at a time, in the
        // place of the queries; then a warp has 8 of the channels, a lane a row.
        float* join_s = reinterpret_cast<float*>(q_s);   // [group and copy][64 channels][row of the copy]
        const int state = g * copies + copy;
        if (warp_live) ml_s[state * copy_rows + row % copy_rows] = make_float2(m, l);
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          // (the queries may go once both groups' scores are there; the half before, once all have read it)
          if (h == 0) {
            __syncwarp();
            if (lane == 0) mbar_arrive(X_FREE);
          }
          if (!wait_for(X_FREE, frees++ & 1)) break;
          if (warp_live && !fresh) {
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t o[32];
              tmem_ld_x32(O + 64 * h + 32 * c, o);
              tmem_wait_ld();
              float* to = join_s + (state * 64 + 32 * c) * copy_rows + row % copy_rows;
#pragma unroll
              for (int e = 0; e < 32; ++e) to[e * copy_rows] = __uint_as_float(o[e]) * scale;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(X_FULL);
          if (!wait_for(X_FULL, fulls++ & 1)) break;
          const int odd_h = h ? odd_1 : odd_0;
#pragma unroll 1
          for (int of_copy = lane; of_copy < rows; of_copy += 32) {
            float2 ml[8];
            float now = PA_NOTHING, sum = 0.f, x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              ml[i] = i < 2 * copies ? ml_s[i * copy_rows + of_copy] : make_float2(PA_NOTHING, 0.f);
              now = fmaxf(now, ml[i].x);
            }
            // (all loads first: what is not there is read and left out)
            const float* from = join_s + 8 * warp * copy_rows + of_copy;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (i >= 2 * copies) break;
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = from[(i * 64 + e) * copy_rows];
              const bool has = ml[i].x != PA_NOTHING || ml[i].y != 0.f;   // (or it saw nothing, or had no tile)
              const float by = has ? ex2(ml[i].x - now) : 0.f;
              sum = fmaf(ml[i].y, by, sum);
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = fmaf(has ? v[e] : 0.f, by, x[e]);
            }
            const int64_t at = row_of(of_copy);
            if (h == 0 && warp == 0) put_sums(at, now, sum);
            const float inv = !finish ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= inv;
            if (odd_h != INT_MAX && odd_h < min(walk.u.pos0 + p.over_ratio(walk.unit * PT_ROWS + of_copy) + 1, room)) {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(0x7fffffffu);
            }
            put8(at, 8 * h + warp, x);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(X_FREE);
        }
        // the next piece's queries go where the others may still be reading
        if (!bad) wait_for(X_FREE, frees++ & 1);
      }
      tc_fence_before();
    }
  }
  if (tid == 0 && *abort_s && p.status) atomicOr(p.status, PG_GAVE_UP);
  tc_fence_before();
  __syncthreads();
  if (warp == PT_MMA_WARP) tmem_dealloc(tmem, 512);
}

// Joins the pieces of the unit that begins in a CTA's run and ends behind it, in order; a warp per row.
template <typename T>
__global__ void __launch_bounds__(256) paged_tile_merge_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int DEPTH = 4;                               // pieces in flight
  griddep_launch();
  griddep_wait();
  const int4 item = p.items[blockIdx.x];
  if (item.x == 0) return;
  const int row = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const PagedSeq seq = paged_seq(p.c, item.x - 1, p.rows);
  const TileUnits u = tile_units(p, seq);
  const int kv = item.y / u.count, cc = (item.y - kv * u.count) * PT_ROWS + row;
  if (cc >= u.cols) return;
  float top = PA_NOTHING, sum = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < item.z; i0 += DEPTH) {
    float2 ml[DEPTH];
    float4 v[DEPTH];
#pragma unroll
    for (int k = 0; k < DEPTH; ++k) {
      const int i = i0 + k;
      const float* rec = p.part + ((2 * (int64_t)(blockIdx.x + i) + (i == 0 ? item.w : 0)) * PT_ROWS + row) * PART;
      ml[k] = i < item.z ? *reinterpret_cast<const float2*>(rec) : make_float2(PA_NOTHING, 0.f);
      v[k] = i < item.z ? *reinterpret_cast<const float4*>(rec + 4 + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < DEPTH; ++k) {
      const float now = fmaxf(top, ml[k].x), old = ex2(top - now), by = ex2(ml[k].x - now);
      top = now;
      sum = fmaf(ml[k].y, by, sum * old);
      a.x = fmaf(v[k].x, by, a.x * old);
      a.y = fmaf(v[k].y, by, a.y * old);
      a.z = fmaf(v[k].z, by, a.z * old);
      a.w = fmaf(v[k].w, by, a.w * old);
    }
  }
  const int tok = p.over_ratio(cc);
  const int64_t out_row = (int64_t)(seq.first + tok) * p.n_q + kv * p.ratio + cc - tok * p.ratio;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>((T*)p.out + out_row * HD + 4 * lane) = make_uint2(Pair<T>::put(a.x * inv, a.y * inv), Pair<T>::put(a.z * inv, a.w * inv));
  if (p.lse && lane == 0) p.lse[out_row] = sum == 0.f ? neg_inf() : (top + log2f(sum)) * LN2;
}

static int tile_ctas() { return sm_count() > 0 ? sm_count() : 1; }
static size_t tile_items_bytes() { return ((size_t)tile_ctas() * sizeof(int4) + 127) & ~(size_t)127; }

size_t paged_tile_bytes() { return tile_items_bytes() + (size_t)2 * tile_ctas() * PT_ROWS * PART * 4; }

template <typename T>
static cudaError_t launch_tile(const PagedAttnParams& p, cudaStream_t st) {
  static std::atomic<bool> configured[MAX_DEVICES];
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= MAX_DEVICES) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(paged_tile_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, PT_SMEM);
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(tile_ctas());
  cfg.blockDim = dim3(PT_THREADS);
  cfg.dynamicSmemBytes = PT_SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, paged_tile_kernel<T>, p);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(tile_ctas(), PT_ROWS / 8);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_tile_merge_kernel<T>, p);
}

cudaError_t launch_paged_tile(const PagedAttnParams& params, bool bf16, void* workspace, cudaStream_t st) {
  PagedAttnParams p = params;
  p.items = (int4*)workspace;
  p.part = (float*)((unsigned char*)workspace + tile_items_bytes());
  return bf16 ? launch_tile<__nv_bfloat16>(p, st) : launch_tile<__half>(p, st);
}

}  // namespace shard
