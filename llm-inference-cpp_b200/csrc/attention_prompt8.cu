// Attention of prompts over the paged cache held in 8 bits (rows8.cuh) on the 5th-generation tensor cores (tcgen05), bf16 queries,
// head size 64 or 128.  For a row at position p of kv head g, over the keys j of its sequence it sees:
//     s_j = scale * k_scale[j] * (q . k_code[j]),   w = softmax(s),   out = sum_j w_j * v_scale[j] * v_code[j]
// (reference loop: src/model/transformer.cpp:263-282.)
//
// A block takes 256 query rows of one sequence and kv head — tokens times the heads of the group, token by token, so that a page
// serves the whole group — as two tiles of 128 rows, and walks the pages (64 keys) that they see:
//
//   scales        a warp makes each row's factor of the page (three of them, for a page a stage each)
//   codes -> fp16 four warps bring a page's codes into a ring with cp.async, each thread what it will read itself, so that nobody waits
//                 for anybody (a thread that asks for bulk copies is busy half a microsecond with each: four a page were 2,000 clocks,
//                 most of a page's time), and make K' = code * (k_scale / kmax) and V' = code * (v_scale / vmax) of a page, kmax and
//                 vmax its largest scales, rounded to fp16 once (half a step is 2^-11 of a number; a bf16 cache's is 2^-8), in the
//                 swizzled layout that the products read; so the scales cost the softmax nothing per key: kmax joins its scale,
//                 log2 vmax its offset.  (A page whose scales are more than 2^12 apart would lose bits of its small rows, which may be
//                 all that a query sees: there K' and V' are the codes themselves and the softmax takes each key's scales.)
//   S = Q' K'^T   tcgen05.mma, Q' the queries times a power of two per row that brings its largest near 2^15, in fp16: bf16 queries
//                 exactly, down to 2^-29 of the row's largest entry; 32-bit ones (those that `rope` makes, which every layer of a
//                 model passes) rounded to 11 bits, as the keys are: kept as two fp16 numbers they would double the products, for an
//                 output that is rounded to bf16
//   softmax       two threads own a row, 32 keys of a page each: tcgen05.ld, mask, maximum, exp2, sum; P = 2^(s + log2 vmax - m) goes
//                 back to tensor memory as fp16 over the S it has read; the sum of w is that of P / vmax
//   O += P V'     tcgen05.mma with A in tensor memory, accumulating in fp32; m lies 7 below the running maximum (of s + log2 vmax)
//                 and follows it only when that has grown by more than 8, so O is rescaled a few times per row.  P is at most 2^15
//                 and for the largest 2^7 or more: it keeps 11 bits down to 2^-21 of the row's largest, and what is below is off by
//                 2^-32 of that at most (with m at the maximum itself 32,000 keys 17.5 nats below another were lost together: 8e-4 of
//                 the output).  At head size 64 tensor memory has room for
//                 an O of each thread's keys, with their own m and sum: nothing passes between the two before the end.  At 128 the two
//                 share one O, ask each other on every page whether an m has to follow (a barrier of 64 threads, 7 % of the page at 64),
//                 and exchange maxima only then.
//
// What bounds it: a row's way through the softmax of a page, 1,800 clocks from S to P with four warps on each scheduler; the
// exponentials alone (16 a clock and SM) are 1,024 for the two tiles, the products 256 at head size 64 and 512 at 128, the
// conversion 700 and 1,300 beside them.  A page of two tiles takes 1,900 and 2,400 clocks.  Measured: 2,048 tokens, 32 heads of 64,
// 52 us (331 TFLOP/s); 600 and 600 tokens over 20,011 to 31,001 positions, 32 heads by 8 of 128, 589 us (664 TFLOP/s, 0.41 of what a
// library's bf16 product reaches).
//
// A step of few blocks leaves SMs idle: then a block's pages are cut into parts, each a block of its own that leaves (m, sum, O) per
// row in a workspace; a second kernel joins them in order.  Waits are bounded (sm100.cuh).
#include <math.h>

#include <type_traits>

#include "mma_sync.cuh"
#include "rows8.cuh"
#include "tc_common.cuh"

namespace llmi {

constexpr int P8_ROWS = 256, P8_TILE = 128;
// Warps: 0, 2, 3 scales, 1 products, 4 .. 19 softmax (two tiles, two halves of a page's keys, four quarters of the rows),
// 20 .. 23 codes to fp16.
constexpr int P8_SOFTMAX = 4, P8_CONVERT = 20, P8_WARPS = 24;
constexpr int P8_THREADS = P8_WARPS * 32;
constexpr int P8_JOINS = 32;              // blocks of 8 warps that join a block's rows
constexpr int P8_TMEM = 512;              // per tile of rows 256 columns: S of even and odd pages (64 each), O (D, or 64 of each half of the keys)
constexpr float P8_UP = 7.0f;             // where the reference maximum moves it goes 7 below the largest score: weights of up to 2^7
constexpr float P8_LAZY = 15.0f;          // it moves where a weight would pass 2^15
constexpr uint32_t PG_WIDE = 1u, PG_POISON = 2u;       // the page's scales are far apart; it has values that are no numbers
constexpr float P8_LIGHT = 8.077935669463161e-28f;     // 2^-90
constexpr float P8_APART = 2.44140625e-4f;             // 2^-12
constexpr float P8_TINY = 7.888609052210118e-31f;      // 2^-100: smaller scales of a page count as this
constexpr float P8_MUCH = 5.192296858534828e33f;       // 2^112: sums of weights beyond this move the reference, too (values near 2^-100)

struct Prompt8Params {
  const void* q;                // bf16, or fp32 with q_f32
  long ldq;
  __nv_bfloat16* out;
  long ldo;
  const uint8_t* k_codes;
  const float* k_scales;
  const uint8_t* v_codes;
  const float* v_scales;
  const int32_t* seq_q_start;   // [n_seqs + 1]
  const int32_t* seq_kv_len;    // [n_seqs]
  Paged8 kv;
  int n_seqs, group;
  float scale_log2;
  int window;
  int q_f32;
  int parts, part_pages;        // most parts of a block's pages; the least pages of a part
  float* partials;              // [block][kv head][part][256][D + 2] when parts > 1
  int* error_flag;
};

template <int D>
struct P8Cfg {
  static constexpr int SUBS = D / 64;                     // 64-column sub-tiles of a row
  static constexpr bool OWN = D == 64;                    // each of a row's two threads has a maximum, a sum and an O of its own
  static constexpr int Q_TILE = SUBS * P8_TILE * 128;     // bytes of a tile's queries
  static constexpr int KV_TILE = SUBS * PAGE8 * 128;      // bytes of a page's K' or V'
  static constexpr int STAGE = 2 * KV_TILE, STAGES = 3;
  static constexpr int RAW = 2 * PAGE8 * D, RAWS = D == 64 ? 4 : 3;      // codes of a page; pages under way
  static constexpr int SMEM = 1024 + 2 * Q_TILE + STAGES * STAGE + RAWS * RAW + 176;
};

// Block b of the step's blocks of 256 rows, counted from the last block of the last sequence backwards (late blocks see more keys and
// come first).  A whole warp calls this.
struct P8Block {
  int seq, q_start, row0, rows, pos0, first, last, lo, pg_first, n_pages;      // rows 0: there is no such block
};
__device__ __forceinline__ P8Block prompt8_block(const Prompt8Params& p, int b) {
  const int lane = threadIdx.x & 31;
  P8Block d;
  d.rows = d.n_pages = 0;
  for (int s0 = p.n_seqs - 1; s0 >= 0; s0 -= 32) {
    const int s = s0 - lane;
    int start = 0, q_len = 0, kv_len = 0;
    if (s >= 0) start = p.seq_q_start[s], q_len = p.seq_q_start[s + 1] - start, kv_len = p.seq_kv_len[s];
    const int n = kv_len > 0 ? (q_len * p.group + P8_ROWS - 1) / P8_ROWS : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int all = __shfl_sync(0xffffffffu, x, 31);
    if (b < all) {
      const int src = __ffs(__ballot_sync(0xffffffffu, x > b)) - 1;
      d.seq = s0 - src;
      const int mb = __shfl_sync(0xffffffffu, x, src) - 1 - b;
      d.q_start = __shfl_sync(0xffffffffu, start, src);
      q_len = __shfl_sync(0xffffffffu, q_len, src);
      kv_len = __shfl_sync(0xffffffffu, kv_len, src);
      d.row0 = mb * P8_ROWS;
      d.rows = min(P8_ROWS, q_len * p.group - d.row0);
      d.pos0 = kv_len - q_len;
      d.first = d.pos0 + d.row0 / p.group;
      d.last = d.pos0 + (d.row0 + d.rows - 1) / p.group;
      d.lo = (p.window > 0 && d.first - p.window + 1 > 0) ? d.first - p.window + 1 : 0;
      d.pg_first = page_index8(p.kv, d.lo);
      if (d.last >= 0) d.n_pages = page_index8(p.kv, d.last) - d.pg_first + 1;
      return d;
    }
    b -= all;
  }
  return d;
}
// Its pages in parts of equal size: (parts, pages of one).
__device__ __forceinline__ int2 prompt8_parts(const Prompt8Params& p, int n_pages) {
  const int n = max(1, min(p.parts, n_pages / p.part_pages));
  const int per = max(1, (n_pages + n - 1) / n);
  return make_int2(max(1, (n_pages + per - 1) / per), per);
}

// 16 columns of this thread's TMEM lane; no wait
__device__ __forceinline__ void p8_ld16(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void p8_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void p8_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void p8_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Products and commits by the one lane of a warp that has `one` set; the whole warp comes here, so that descriptors and addresses stay
// in uniform registers (in a branch of one lane each product's way there took 65 clocks, 2.4 of the 3.5 thousand a page at D = 128).
__device__ __forceinline__ void p8_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(one)
      : "memory");
}
__device__ __forceinline__ void p8_mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc), "r"(one)
      : "memory");
}
__device__ __forceinline__ void p8_commit(uint32_t bar, uint32_t one) {
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
               ::"r"(bar), "r"(one) : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }

template <int D, int HELD>
__global__ void __launch_bounds__(P8_THREADS, 1) attention_prompt8_kernel(Prompt8Params p) {
  using C = P8Cfg<D>;
  constexpr int STAGES = C::STAGES, RAWS = C::RAWS;
  constexpr bool OWN = C::OWN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const base_p = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_smem = base, kv_smem = q_smem + 2 * C::Q_TILE, raw_smem = kv_smem + STAGES * C::STAGE, bars = raw_smem + RAWS * C::RAW;
  const uint32_t q_full = bars, tmem_slot = bars + 168;
  auto fac_full = [&](int s) { return bars + 8u * (1 + s); };
  auto kv_full = [&](int s) { return bars + 8u * (1 + STAGES + s); };
  auto kv_empty = [&](int s) { return bars + 8u * (1 + 2 * STAGES + s); };
  auto s_full = [&](int tile, int b) { return bars + 8u * (1 + 3 * STAGES + 2 * tile + b); };
  auto p_ready = [&](int tile, int b) { return bars + 8u * (5 + 3 * STAGES + 2 * tile + b); };
  auto o_done = [&](int tile) { return bars + 8u * (9 + 3 * STAGES + tile); };
  static_assert(8 * (11 + 3 * STAGES) <= 168, "barriers fit");
  __shared__ float s_scales[STAGES][2][2 * PAGE8];       // pages under way: scales of keys, of values
  __shared__ uint2 s_fac[STAGES][PAGE8];                 // a row's factors, each the sum of two fp16 numbers: of its keys, of its values
  __shared__ uint32_t s_none[STAGES][4];                 // rows whose key codes, and whose value codes, may be no numbers
  __shared__ float4 s_page[STAGES];                      // kmax, log2 vmax, 1 / vmax, whether the page needs a look (PG_*, as bits)
  __shared__ uint32_t s_poison[STAGES][2];               // keys whose values are no numbers
  __shared__ float s_top[2][2][P8_TILE];                 // [tile][half][row]: the largest score of a row's half
  __shared__ float s_sum[2][2][P8_TILE];
  __shared__ float s_key[STAGES][2][PAGE8];              // k_scale, log2 v_scale

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x, G = p.group, Hkv = p.kv.n_kv_heads;
  const int blk = blockIdx.y / p.parts, part = blockIdx.y % p.parts;
  const P8Block d = prompt8_block(p, blk);               // (of the step's index block)
  const int2 cut = prompt8_parts(p, d.n_pages);
  const int v0 = part * cut.y, n_pg = min(cut.y, d.n_pages - v0);
  // (no such block or part; positions below 0 only: nothing to see)
  if (d.rows <= 0 || part >= cut.x || n_pg <= 0) {
    pdl_wait();
    return;
  }
  const int pg0 = d.pg_first + v0;                       // this part's first page
  // pages of this part that a tile's rows see the first key of
  int n_tile[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int rows = min(P8_TILE, d.rows - i * P8_TILE);
    n_tile[i] = 0;
    if (rows > 0) {
      const int last = d.pos0 + (d.row0 + i * P8_TILE + rows - 1) / G;
      if (last >= 0) n_tile[i] = max(0, min(n_pg, last / PAGE8 - pg0 + 1));
    }
  }

  if (threadIdx.x == 0) {
    mbar_init(q_full, 16);
    for (int s = 0; s < STAGES; ++s) mbar_init(fac_full(s), 1), mbar_init(kv_full(s), 4), mbar_init(kv_empty(s), 1);
    for (int i = 0; i < 2; ++i) {
      for (int b = 0; b < 2; ++b) mbar_init(s_full(i, b), 1), mbar_init(p_ready(i, b), 8);
      mbar_init(o_done(i), 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(P8_TMEM));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  pdl_wait();
  pdl_launch_dependents();      // (not ahead of the tensor memory: a kernel behind this one could take it and wait for this block)

  // the page of the pool that page j of this part is, or -1
  const int32_t* table = p.kv.seq_pages + (size_t)d.seq * p.kv.pages_stride;
  auto page_at = [&](int j) {
    const int at = pg0 + j, page = j < n_pg && at < p.kv.table_pages ? table[at] : -1;
    return (unsigned)page < (unsigned)p.kv.n_pages ? page : -1;
  };
  const int scale_stage = warp == 0 ? 0 : warp - 1;      // (of the warps 0, 2 and 3)
  if (warp < P8_SOFTMAX && warp != 1) {
    // ---- scales: what the softmax needs of a page, and its rows' factors; a warp for each of the three stages ----
    static_assert(STAGES == 3, "warps 0, 2 and 3");
    const int st = scale_stage;
    auto ask = [&](int j) {                                        // lanes 0 .. 15: the keys' scales, the others: the values'
      const int page = page_at(j);
      const size_t row = ((size_t)max(page, 0) * Hkv + kvh) * PAGE8 + (lane & 15) * 4;
      cp_async16(&s_scales[st][(j / STAGES) & 1][lane * 4], (lane < 16 ? p.k_scales : p.v_scales) + row, 16);
      cp_async_commit();
      return page;
    };
    int page = ask(st);
    uint32_t phase = 1u;
    for (int j = st; j < n_pg; j += STAGES, phase ^= 1u) {
      const bool known = page >= 0;
      page = ask(j + STAGES);
      cp_async_wait<1>();
      __syncwarp();
      const float* ks = s_scales[st][(j / STAGES) & 1];
      const int a = max(d.lo - (pg0 + j) * PAGE8, 0), b = min(d.last - (pg0 + j) * PAGE8, 63);      // rows that some query sees
      // the page's largest scales (of rows that are numbers), the least but zeros, and its rows that are no numbers
      float x[2], y[2], km = 0.f, vm = 0.f, kn = INFINITY, vn = INFINITY;
      uint32_t bad[2], out[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = lane + 32 * h;
        const bool in = r >= a && r <= b;
        x[h] = in && known ? ks[r] : 0.f;
        y[h] = in ? (known ? ks[PAGE8 + r] : __int_as_float(0x7fffffff)) : 0.f;
        const float fx = finite8(x[h]) ? fabsf(x[h]) : 0.f, fy = finite8(y[h]) ? fabsf(y[h]) : 0.f;
        km = fmaxf(km, fx), vm = fmaxf(vm, fy);
        if (fx != 0.f) kn = fminf(kn, fx);
        if (fy != 0.f) vn = fminf(vn, fy);
        bad[h] = __ballot_sync(0xffffffffu, !finite8(y[h]));
        out[h] = __ballot_sync(0xffffffffu, !(in && known));
      }
      // (numbers that are not negative are ordered as their bits are)
      km = fmaxf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(km))), P8_TINY);
      vm = fmaxf(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(vm))), P8_TINY);
      const bool wide = __any_sync(0xffffffffu, kn < km * P8_APART || vn < vm * P8_APART);
      const float k_inv = __frcp_rn(km), v_inv = __frcp_rn(vm), lv = wide ? 0.f : fast_log2(vm);
      // (the softmax is done with what is there of the page three before)
      if (j >= STAGES && !mbar_wait(kv_empty(st), phase, p.error_flag, 109)) break;
      if (lane == 0) {
        s_page[st] = make_float4(km, lv, v_inv, __uint_as_float((wide ? PG_WIDE : 0u) | ((bad[0] | bad[1]) ? PG_POISON : 0u)));
        s_poison[st][0] = bad[0];
        s_poison[st][1] = bad[1];
        s_none[st][0] = out[0], s_none[st][1] = out[1], s_none[st][2] = out[0] | bad[0], s_none[st][3] = out[1] | bad[1];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = lane + 32 * h;
        float kf = x[h] * k_inv, vf = finite8(y[h]) ? y[h] * v_inv : 0.f;
        if (wide) {
          const float own = fmaxf(y[h], P8_TINY);                          // (a NaN's values are zeros here: its bit is in s_poison)
          s_key[st][0][r] = x[h];
          s_key[st][1][r] = log2f(own);
          kf = 1.f;
          vf = finite8(y[h]) ? y[h] / own : 0.f;
        }
        const __half kh = __float2half_rn(kf), vh = __float2half_rn(vf);
        s_fac[st][r] = make_uint2(half2_bits(__halves2half2(kh, __float2half_rn(kf - __half2float(kh)))),
                                 half2_bits(__halves2half2(vh, __float2half_rn(vf - __half2float(vh)))));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(fac_full(st));
    }
    cp_async_wait_all();
  } else if (warp == 1) {
    // ---- products ----
    // S: A = Q' (K-major), B = K' (K-major), 64 columns; O: A = P (tensor memory, 32 columns of fp16 pairs), B = V' (MN-major, sub-tiles
    // of 64 dims KV_TILE / SUBS apart).  MMAs of one thread run in issue order: S_{j+1} may be issued into the buffer that P_{j-1} lies in
    // once O += P_{j-1} V_{j-1} was.  Everything here is the same in all lanes.
    const uint32_t idesc_s = (1u << 4) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    const uint32_t one = elect_one(), tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int pages = __shfl_sync(0xffffffffu, n_pg, 0);
    const int in_tile[2] = {__shfl_sync(0xffffffffu, n_tile[0], 0), __shfl_sync(0xffffffffu, n_tile[1], 0)};
    const uint64_t desc_q = umma_desc(q_smem);
    const uint64_t desc_k = umma_desc(kv_smem);
    const uint64_t desc_v = umma_desc(kv_smem + C::KV_TILE) + ((uint64_t)((PAGE8 * 128 >> 4) - 1) << 16);      // leading offset: to the next 64 dims
    auto issue_s = [&](int tile, int j, int st) {
      const uint32_t dst = tm + 256u * tile + 64u * (j & 1);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
        p8_mma(dst, desc_q + (uint32_t)((tile * C::Q_TILE + (k / 4) * (P8_TILE * 128)) >> 4) + 2 * (k % 4),
               desc_k + (uint32_t)(st * (C::STAGE >> 4)) + ((k / 4) * (PAGE8 * 128) >> 4) + 2 * (k % 4), idesc_s, k > 0, one);
      p8_commit(s_full(tile, j & 1), one);
    };
    auto issue_o = [&](int tile, int j, int st) {
      const uint32_t a = tm + 256u * tile + 64u * (j & 1), o = tm + 256u * tile + 128u;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        p8_mma_ts(OWN ? o + 64u * (k / 2) : o, a + 32u * (k / 2) + 8u * (k % 2), desc_v + (uint32_t)(st * (C::STAGE >> 4)) + (k * (16 * 128) >> 4), idesc_o,
                  (j > 0 || (OWN ? k % 2 : k) > 0) ? 1u : 0u, one);
      p8_commit(o_done(tile), one);
    };
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, p.error_flag, 102));
    int st = 0, before = 0;              // the stage of page j, of page j - 1
    uint32_t phase = 0;
    for (int j = 0; j <= pages && ok; ++j) {
      if (j < pages) {
        ok = __all_sync(0xffffffffu, mbar_wait(kv_full(st), phase, p.error_flag, 103));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int tile = 0; tile < 2; ++tile)
          if (j < in_tile[tile]) issue_s(tile, j, st);
      }
      if (j >= 1) {
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          if (j - 1 >= in_tile[tile] || !ok) continue;
          ok = __all_sync(0xffffffffu, mbar_wait(p_ready(tile, (j - 1) & 1), ((j - 1) >> 1) & 1, p.error_flag, 104));
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (ok) issue_o(tile, j - 1, before);
        }
        if (j - 1 + STAGES < pages) p8_commit(kv_empty(before), one);      // (where the stage is filled again)
      }
      before = st;
      if (++st == STAGES) st = 0, phase ^= 1u;
    }
  } else if (warp >= P8_SOFTMAX && warp < P8_CONVERT) {
    // ---- softmax and output: two threads a row, each with 32 keys of every page and half of the row's output ----
    constexpr int HD = D / 2, OC = OWN ? D : HD;                   // OC: columns of O that a thread rescales
    const int tile = (warp - P8_SOFTMAX) >> 3, half = ((warp - P8_SOFTMAX) >> 2) & 1, quad = warp & 3;
    const int in_tile = quad * 32 + lane, r = tile * P8_TILE + in_tile;       // the row's TMEM lane, the row of the block
    const int row = d.row0 + r, tok = row / G, head = kvh * G + row % G;
    const bool row_ok = r < d.rows;
    const int qpos = d.pos0 + (d.row0 + min(r, d.rows - 1)) / G;
    const int pos_a = __shfl_sync(0xffffffffu, qpos, 0), pos_b = __shfl_sync(0xffffffffu, qpos, 31);      // the warp's first and last
    // what the two threads of a row tell each other: 64 threads meet
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + tile * 4 + quad) : "memory"); };
    auto any_of_pair = [&](bool x) {
      uint32_t r;
      asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                   : "=r"(r) : "r"(1 + tile * 4 + quad), "r"(x ? 1u : 0u) : "memory");
      return r != 0u;
    };
    // The rows' queries, times a power of two each.  The two warps of 32 rows take 16 each, the lanes of a row
    // beside each other, with a row's 8 entries a lane and BATCH loads under way.
    float row_fac;
    {
      constexpr int LANES = D / 8, AT_ONCE = 32 / LANES, BATCH = 4;
      const int c = lane % LANES;
      auto queries = [&](auto f32) {
#pragma unroll 1
        for (int r0 = quad * 32 + half * 16; r0 < quad * 32 + half * 16 + 16; r0 += BATCH * AT_ONCE) {
          uint4 raw[BATCH][decltype(f32)::value ? 2 : 1];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int r2 = tile * P8_TILE + r0 + i * AT_ONCE + lane / LANES, row2 = d.row0 + r2;
            const size_t src = (size_t)(d.q_start + row2 / G) * p.ldq + (size_t)(kvh * G + row2 % G) * D + 8 * c;
            const uint4* from = decltype(f32)::value ? reinterpret_cast<const uint4*>((const float*)p.q + src) : reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.q + src);
#pragma unroll
            for (int u = 0; u < (decltype(f32)::value ? 2 : 1); ++u) raw[i][u] = r2 < d.rows ? from[u] : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int in = r0 + i * AT_ONCE + lane / LANES;
            float x[8];
            if (decltype(f32)::value) {
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const uint4 w = raw[i][decltype(f32)::value ? u : 0];
                x[4 * u] = __uint_as_float(w.x), x[4 * u + 1] = __uint_as_float(w.y), x[4 * u + 2] = __uint_as_float(w.z), x[4 * u + 3] = __uint_as_float(w.w);
              }
            } else {
              const uint32_t w[4] = {raw[i][0].x, raw[i][0].y, raw[i][0].z, raw[i][0].w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                x[2 * e] = __uint_as_float(w[e] << 16);
                x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
              }
            }
            float a = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(x[e]));
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            // the row's largest entry lies between 2^14 and 2^15 (rows that are zero or not finite: as they are, times 2^15)
            int up = 15;
            if (a > 0.f && a <= FLT_MAX) up = min(115, 141 - (int)(__float_as_uint(a) >> 23));
            float down = __uint_as_float((uint32_t)(127 + up) << 23);
            if (p.scale_log2 < 0.f) down = -down;                  // the factor of the scores below is positive
            if (c == 0) s_top[tile][0][in] = ldexpf(fabsf(p.scale_log2), -up);
            uint32_t h[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = half2_bits(__floats2half2_rn(x[2 * e] * down, x[2 * e + 1] * down));
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};"
                         ::"r"(q_smem + tile * C::Q_TILE + in * 128 + (c / 8) * (P8_TILE * 128) + (((c % 8) ^ (in & 7)) << 4)),
                         "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
          }
        }
      };
      if (p.q_f32) queries(std::true_type{});
      else queries(std::false_type{});
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      meet();
      row_fac = s_top[tile][0][in_tile];
    }
    const int n = n_tile[tile];
    const uint32_t t_lane = (uint32_t)(quad * 32) << 16, t_tile = tmem + 256u * tile + t_lane, t_o = t_tile + 128u + (uint32_t)(OC * half);
    // the reference (7 below a maximum of s + log2 vmax, base 2) and 0 less it (0 while there is none); the sum of 2^(s - m_ref) over this half, and
    // (where the halves share a maximum) over the other one when they last met
    float m_ref = -INFINITY, neg_ref = 0.f, l_run = 0.f, l_other = 0.f;
    bool ok = true;
    int st = 0;                                                    // j % STAGES
    // (after a wait that gave up the pages are gone through without waiting: the two threads of a row go on meeting)
    for (int j = 0; j < n; ++j, st = st + 1 == STAGES ? 0 : st + 1) {
      ok = ok && mbar_wait(s_full(tile, j & 1), (j >> 1) & 1, p.error_flag, 105);
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t t_s = t_tile + 64u * (j & 1) + 32u * half;    // this half's scores, then its weights
      float sc[32];
      p8_ld16(t_s, sc);
      p8_ld16(t_s + 16u, sc + 16);
      const float4 page = s_page[st];
      const uint32_t look = __float_as_uint(page.w);
      const int key0 = (pg0 + j) * PAGE8 + 32 * half;
      // (never 0, where small queries meet small keys: 0 times a masked key's -inf is no number)
      float to_log2 = fmaxf(row_fac * page.x, FLT_MIN), off = page.y + neg_ref;
      p8_ld_wait();
      if (look & PG_WIDE) {                                        // (kmax 1 / row_fac, vmax 1: the scores are final)
        to_log2 = 1.f;
#pragma unroll
        for (int c = 0; c < 32; ++c) sc[c] = fmaf(sc[c], row_fac * s_key[st][0][32 * half + c], s_key[st][1][32 * half + c]);
      }
      if (key0 + 31 > pos_a || (p.window > 0 && key0 <= pos_b - p.window)) {
        const int a = p.window > 0 ? qpos - p.window + 1 - key0 : 0, b = qpos - key0;      // the keys a .. b are seen
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if (c > b || c < a) sc[c] = -INFINITY;
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 32; c += 8)
#pragma unroll
        for (int u = 0; u < 4; ++u) mx4[u] = fmaxf(fmaxf(mx4[u], sc[c + 2 * u]), sc[c + 2 * u + 1]);
      float top = fmaf(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), to_log2, page.y), corr = 1.f;
      // The common page: nothing has outgrown the reference maximum, and the sum of w is that of P / vmax.  Otherwise all threads of
      // the warp, or of the two that share rows and their Os, go the long way.
      const bool light = look != 0u || page.z * P8_LIGHT > l_run + l_other;
      bool by_key = false;
      const bool grown = top > m_ref + P8_LAZY || light || l_run > P8_MUCH;
      if (OWN ? __any_sync(0xffffffffu, grown) : any_of_pair(grown)) {
        if (!OWN) {
          s_top[tile][half][in_tile] = top;
          s_sum[tile][half][in_tile] = l_run;
          meet();
          top = fmaxf(top, s_top[tile][half ^ 1][in_tile]);
          l_other = s_sum[tile][half ^ 1][in_tile];
          meet();
        }
        const bool much = l_run + l_other > P8_MUCH;
        if (top > m_ref + P8_LAZY || much) {
          top = fmaxf(top - P8_UP, much ? m_ref + P8_LAZY : -INFINITY);
          if (m_ref != -INFINITY) {
            corr = fast_exp2(m_ref - top);
            l_run = rescale8(l_run, m_ref - top);
            l_other = rescale8(l_other, m_ref - top);
          }
          m_ref = top;
          neg_ref = -top;
        }
        off = page.y + neg_ref;
        by_key = __any_sync(0xffffffffu, look != 0u || page.z * P8_LIGHT > l_run + l_other);
        if (by_key) {
          // The sum of w key by key where P may have lost some of it: in a page whose values are far smaller than another page's (zeros,
          // for instance, say nothing about their weights).
          const bool wide = (look & PG_WIDE) != 0u;
#pragma unroll
          for (int c = 0; c < 32; ++c) l_run += fast_exp2(fmaf(sc[c], to_log2, off) - (wide ? s_key[st][1][32 * half + c] : page.y));
          const uint32_t bad = s_poison[st][half];
          if (bad) {                                               // values that are no numbers: for the rows that see them
            const int a = p.window > 0 ? max(qpos - p.window + 1 - key0, 0) : 0, b = min(qpos - key0, 31);
            if (a <= b && ((bad >> a) << (31 - (b - a)))) l_run = __int_as_float(0x7fffffff);
          }
        }
      }
      const float2 scale2 = make_float2(to_log2, to_log2), off2 = make_float2(off, off);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const float2 x = __ffma2_rn(make_float2(sc[c], sc[c + 1]), scale2, off2);
        sc[c] = x.x, sc[c + 1] = x.y;
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) sc[c] = fast_exp2(sc[c]);
      uint32_t packed[16];
      float2 sum2[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        sum2[(c >> 1) & 3] = __fadd2_rn(sum2[(c >> 1) & 3], make_float2(sc[c], sc[c + 1]));
        packed[c >> 1] = half2_bits(__floats2half2_rn(sc[c], sc[c + 1]));
      }
      if (!by_key) {
        const float2 s = __fadd2_rn(__fadd2_rn(sum2[0], sum2[1]), __fadd2_rn(sum2[2], sum2[3]));
        l_run = fmaf(s.x + s.y, page.z, l_run);
      }
      if (j >= 1) {
        // (waited for on every page: a wait on a phase's parity is right only for a thread at most one phase behind)
        ok = ok && mbar_wait(o_done(tile), (j - 1) & 1, p.error_flag, 106);
        __syncwarp();
        if (__any_sync(0xffffffffu, corr != 1.f)) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
          for (int c = 0; c < OC; c += 16) {
            float t[16];
            uint32_t u[16];
            p8_ld16(t_o + (uint32_t)c, t);
            p8_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(t[e] * corr);
            p8_st16(t_o + (uint32_t)c, u);
          }
        }
      }
      p8_st16(t_s, packed);
      p8_st_wait();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready(tile, j & 1));
    }
    // (`fine` is the same in all lanes: the TMEM loads are the whole warp's)
    const bool fine = __all_sync(0xffffffffu, ok && (n == 0 || mbar_wait(o_done(tile), (n - 1) & 1, p.error_flag, 107)));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // the row's maximum and sum, and what its two Os count for (only where each half has its own)
    s_top[tile][half][in_tile] = m_ref;
    s_sum[tile][half][in_tile] = l_run;
    meet();
    const float m2[2] = {s_top[tile][0][in_tile], s_top[tile][1][in_tile]}, l2[2] = {s_sum[tile][0][in_tile], s_sum[tile][1][in_tile]};
    const float m_all = OWN ? fmaxf(m2[0], m2[1]) : m_ref;
    const float down0 = !OWN || m2[0] == -INFINITY ? 0.f : m2[0] - m_all, down1 = !OWN || m2[1] == -INFINITY ? 0.f : m2[1] - m_all;
    const float l_all = OWN ? rescale8(l2[0], down0) + rescale8(l2[1], down1) : l2[0] + l2[1];
    const float part0 = fast_exp2(down0), part1 = fast_exp2(down1);
    auto output = [&](int c, float (&o)[16]) {                     // dims HD * half + c .. + 15 (zeros without a page)
      if (n == 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = 0.f;
        return;
      }
      p8_ld16(t_tile + 128u + (uint32_t)(HD * half + c), o);
      if (OWN) {
        float other[16];
        p8_ld16(t_tile + 128u + (uint32_t)(D + HD * half + c), other);
        p8_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = fmaf(other[e], part1, o[e] * part0);
      } else {
        p8_ld_wait();
      }
    };
    if (fine) {
      if (cut.x > 1) {
        float* slot = p.partials + (((size_t)blk * Hkv + kvh) * p.parts + part) * (P8_ROWS * (D + 2));
        if (row_ok && half == 0) slot[r] = m_all, slot[P8_ROWS + r] = l_all;
        float* dst = slot + 2 * P8_ROWS + (size_t)r * D + HD * half;
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
          float o[16];
          output(c, o);
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            if (row_ok) *reinterpret_cast<float4*>(dst + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      } else {
        // (a position below 0 sees nothing: zeros; scores that are all -infinity: NaN)
        const float inv = qpos < 0 ? 0.f : 1.f / l_all;
        __nv_bfloat16* dst = p.out + (size_t)(d.q_start + tok) * p.ldo + (size_t)head * D + HD * half;
#pragma unroll 1
        for (int c = 0; c < HD; c += 16) {
          float o[16];
          output(c, o);
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * e] * inv, o[2 * e + 1] * inv);
            w[e] = *reinterpret_cast<uint32_t*>(&h);
          }
          if (row_ok) {
            *reinterpret_cast<uint4*>(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
      }
    }
  } else if (warp >= P8_CONVERT) {
    // ---- codes to fp16 ----
    const int id = threadIdx.x - P8_CONVERT * 32;                          // 0 .. 127
    constexpr int UPR = D / 16, UNITS = PAGE8 * UPR / 128;         // 16-byte pieces of a row, and of a tile per thread
    int next = page_at(0), slot = 0;                               // the slot of the ring filled next
    auto ask = [&](int j) {
      const int page = next;
      next = page_at(j + 1);
      uint8_t* raw = base_p + (raw_smem - base) + slot * C::RAW;
      const size_t row = ((size_t)max(page, 0) * Hkv + kvh) * PAGE8 * D;
#pragma unroll
      for (int i = 0; i < UNITS; ++i) {
        const int x = (id + 128 * i) * 16;
        cp_async16(raw + x, p.k_codes + row + x, page >= 0 ? 16 : 0);
        cp_async16(raw + PAGE8 * D + x, p.v_codes + row + x, page >= 0 ? 16 : 0);
      }
      cp_async_commit();
      slot = slot + 1 == RAWS ? 0 : slot + 1;
    };
#pragma unroll
    for (int i = 0; i < RAWS - 1; ++i) ask(i);
    int st = 0, s = 0;
    uint32_t phase = 0;
    for (int j = 0; j < n_pg; ++j) {
      ask(j + RAWS - 1);                                           // (into the slot that this thread has read last)
      cp_async_wait<RAWS - 1>();
      if (!mbar_wait(fac_full(st), phase, p.error_flag, 110)) break;       // (the stage is free, too)
      const uint8_t* raw = base_p + (raw_smem - base) + s * C::RAW;
      s = s + 1 == RAWS ? 0 : s + 1;
      const uint32_t k_dst = kv_smem + st * C::STAGE, v_dst = k_dst + C::KV_TILE;
      const bool some = HELD == HELD_E4M3 && (s_none[st][2] | s_none[st][3]) != 0u;     // (any int8 code times 0 is 0)
#pragma unroll
      for (int i0 = 0; i0 < UNITS; i0 += 2) {                               // two pieces of keys and of values at a time
        uint4 kw[2], vw[2];
        uint2 f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int x = id + 128 * (i0 + i), r = x / UPR;
          kw[i] = *reinterpret_cast<const uint4*>(raw + x * 16), vw[i] = *reinterpret_cast<const uint4*>(raw + PAGE8 * D + x * 16);
          f[i] = s_fac[st][r];
          if (some) {
            if ((s_none[st][r >> 5] >> (r & 31)) & 1u) kw[i] = make_uint4(0u, 0u, 0u, 0u);
            if ((s_none[st][2 + (r >> 5)] >> (r & 31)) & 1u) vw[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int x = id + 128 * (i0 + i), r = x / UPR, u = x % UPR;
          const __half2 kf = *reinterpret_cast<const __half2*>(&f[i].x), vf = *reinterpret_cast<const __half2*>(&f[i].y);
          const __half2 kh2 = __low2half2(kf), kl2 = __high2half2(kf), vh2 = __low2half2(vf), vl2 = __high2half2(vf);
          const uint32_t* kp = &kw[i].x;
          const uint32_t* vp = &vw[i].x;
          const uint32_t at = (u / 4) * (PAGE8 * 128) + r * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h) {                                     // eight codes: 16 bytes of fp16
            uint32_t kx[4], vx[4];
#pragma unroll
            for (int w = 0; w < 2; ++w) {                                   // a product is rounded once
              uint32_t k0, k1, v0h, v1h;
              halves8x4<HELD>(kp[2 * h + w], k0, k1);
              halves8x4<HELD>(vp[2 * h + w], v0h, v1h);
              kx[2 * w] = half2_bits(__hfma2(bits_half2(k0), kh2, __hmul2(bits_half2(k0), kl2)));
              kx[2 * w + 1] = half2_bits(__hfma2(bits_half2(k1), kh2, __hmul2(bits_half2(k1), kl2)));
              vx[2 * w] = half2_bits(__hfma2(bits_half2(v0h), vh2, __hmul2(bits_half2(v0h), vl2)));
              vx[2 * w + 1] = half2_bits(__hfma2(bits_half2(v1h), vh2, __hmul2(bits_half2(v1h), vl2)));
            }
            const uint32_t o = at + (((2 * (u % 4) + h) ^ (r & 7)) << 4);
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(k_dst + o), "r"(kx[0]), "r"(kx[1]), "r"(kx[2]), "r"(kx[3]));
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(v_dst + o), "r"(vx[0]), "r"(vx[1]), "r"(vx[2]), "r"(vx[3]));
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // the products read what was written
      __syncwarp();
      if (lane == 0) mbar_arrive(kv_full(st));
      if (++st == STAGES) st = 0, phase ^= 1u;
    }
    cp_async_wait_all();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P8_TMEM));
}

// The parts of a block's rows, in order: a warp a row.
template <int D>
__global__ void __launch_bounds__(256) prompt8_join_kernel(Prompt8Params p) {
  const int kvh = blockIdx.x, blk = blockIdx.y / P8_JOINS, lane = threadIdx.x & 31, G = p.group;
  const P8Block d = prompt8_block(p, blk);
  const int2 cut = prompt8_parts(p, d.n_pages);
  pdl_wait();
  pdl_launch_dependents();
  if (d.rows <= 0 || d.n_pages <= 0 || cut.x <= 1) return;
  constexpr int AT_ONCE = 4;               // parts whose sums are under way
  const size_t step = P8_ROWS * (D + 2);
  for (int r = (blockIdx.y % P8_JOINS) * 8 + (threadIdx.x >> 5); r < d.rows; r += 8 * P8_JOINS) {
    const float* slot = p.partials + ((size_t)blk * p.kv.n_kv_heads + kvh) * p.parts * step;
    float ms = -INFINITY, ls = 0.f;                                // of part `lane` (there are 32 at most)
    if (lane < cut.x) ms = slot[lane * step + r], ls = slot[lane * step + P8_ROWS + r];
    float2 x[AT_ONCE][D / 64], o[D / 64];
    auto ask = [&](int z0) {
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const float2* src = reinterpret_cast<const float2*>(slot + min(z0 + i, cut.x - 1) * step + 2 * P8_ROWS + (size_t)r * D);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) x[i][c] = src[lane + 32 * c];
      }
    };
    ask(0);
    const float m = warp_max(ms), down = ms == -INFINITY ? 0.f : ms - m, f = ms == -INFINITY ? 1.f : fast_exp2(ms - m);
    const float l = warp_sum(rescale8(ls, down));
#pragma unroll
    for (int c = 0; c < D / 64; ++c) o[c] = make_float2(0.f, 0.f);
    for (int z0 = 0; z0 < cut.x; z0 += AT_ONCE) {
      if (z0 > 0) ask(z0);
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const float fz = __shfl_sync(0xffffffffu, f, min(z0 + i, 31));
        if (z0 + i < cut.x) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) o[c].x = fmaf(x[i][c].x, fz, o[c].x), o[c].y = fmaf(x[i][c].y, fz, o[c].y);
        }
      }
    }
    const int row = d.row0 + r;
    const float inv = d.pos0 + row / G < 0 ? 0.f : 1.f / l;
    __nv_bfloat162* dst = reinterpret_cast<__nv_bfloat162*>(p.out + (size_t)(d.q_start + row / G) * p.ldo + (size_t)(kvh * G + row % G) * D);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) dst[lane + 32 * c] = __floats2bfloat162_rn(o[c].x * inv, o[c].y * inv);
  }
}

template <int D, int HELD> int launch_prompt8(const Prompt8Params& p, int n_blocks, cudaStream_t stream) {
  static PerDevice<bool> configured;
  if (!configured.here()) {
    if (cudaFuncSetAttribute(attention_prompt8_kernel<D, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize, P8Cfg<D>::SMEM) != cudaSuccess)
      return LLMI_ERR_LAUNCH;
    configured.here() = true;
  }
  const int rc = launch_pdl(PDL_ATTENTION, attention_prompt8_kernel<D, HELD>, dim3((unsigned)p.kv.n_kv_heads, (unsigned)(n_blocks * p.parts)), P8_THREADS,
                            P8Cfg<D>::SMEM, stream, p);
  if (rc != LLMI_OK || p.parts <= 1) return rc;
  return launch_pdl(PDL_ATTENTION, prompt8_join_kernel<D>, dim3((unsigned)p.kv.n_kv_heads, (unsigned)(n_blocks * P8_JOINS)), 256, 0, stream, p);
}

}  // namespace llmi

using namespace llmi;

// `n_blocks`: at least the blocks of 256 rows over all sequences (n_tokens * group / 256 + n_seqs are enough).  `parts` > 1: a block's
// pages in up to so many parts of at least `part_pages` pages, over `partials` of n_blocks * n_kv_heads * parts * 256 * (head_dim + 2)
// floats.
LLMI_EXPORT int llmi_attention_prompt8(int held, const void* q, long ldq, void* out, long ldo, const void* k_codes, const float* k_scales,
                                       const void* v_codes, const float* v_scales, const int32_t* seq_q_start, const int32_t* seq_kv_len,
                                       const int32_t* seq_pages, int pages_stride, int table_pages, int n_seqs, int n_pages, int n_blocks,
                                       int n_heads, int n_kv_heads, int head_dim, float scale, int window, int q_f32, int parts, int part_pages,
                                       float* partials, long n_floats, int* error_flag, cudaStream_t stream) {
  if (n_seqs <= 0 || n_blocks <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || (head_dim != 64 && head_dim != 128) ||
      table_pages <= 0 || n_pages <= 0 || window < 0 || parts <= 0 || part_pages <= 0)
    return LLMI_ERR_BAD_SIZE;
  if ((long)n_blocks * parts > 65535 || parts > 32 || (parts > 1 && n_blocks * P8_JOINS > 65535)) return LLMI_ERR_BAD_SIZE;
  if (parts > 1 && (!partials || n_floats < (long)n_blocks * n_kv_heads * parts * P8_ROWS * (head_dim + 2))) return LLMI_ERR_BAD_SIZE;
  if (held != HELD_INT8 && held != HELD_E4M3) return LLMI_ERR_BAD_DTYPE;
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales | (uintptr_t)partials) & 15) ||
      (ldq & (q_f32 ? 3 : 7)) || (ldo & 7))
    return LLMI_ERR_ALIGN;
  Prompt8Params p{q, ldq, (__nv_bfloat16*)out, ldo, (const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales,
                  seq_q_start, seq_kv_len, Paged8{seq_pages, pages_stride, table_pages, n_pages, n_kv_heads, head_dim}, n_seqs, n_heads / n_kv_heads,
                  scale * 1.4426950408889634f, window, q_f32, parts, part_pages, partials, error_flag};
  if (head_dim == 64) return held == HELD_INT8 ? launch_prompt8<64, HELD_INT8>(p, n_blocks, stream) : launch_prompt8<64, HELD_E4M3>(p, n_blocks, stream);
  return held == HELD_INT8 ? launch_prompt8<128, HELD_INT8>(p, n_blocks, stream) : launch_prompt8<128, HELD_E4M3>(p, n_blocks, stream);
}
