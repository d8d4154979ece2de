// Attention of few query rows a sequence — single tokens, short messages — over the paged cache held in 8 bits (rows8.cuh), bf16
// queries, head size 64 or 128.  For a row at position p of kv head g, over the keys j of its sequence it sees:
//     s_j = scale * k_scale[j] * (q . k_code[j]),   w = softmax(s),   out = sum_j w_j * v_scale[j] * v_code[j]
// (reference loop: src/model/transformer.cpp:263-282).  Every code is read once and takes part in a handful of operations, so what
// bounds the kernel is HBM: 2 (D + 4) bytes a position and kv head.
//
//  * All pages that the step's rows see, kv head by kv head and sequence by sequence, are one line of units (a unit: one page of one
//    kv head), cut into as many equal ranges as there are blocks resident on the device.  A block works through its range whatever
//    the sequences' lengths are, so no block waits for the longest one, and nothing about the cut depends on what the host knows.
//    A (sequence, kv head) whose units several ranges share is joined by the block that comes last (a ticket per kv head and
//    sequence), in the order of the ranges: the same call gives the same bits.
//  * Within a block each warp takes every eighth chunk (2 KB of key codes, 2 KB of value codes, their scales) into a ring of its own
//    in shared memory with cp.async, across the borders of sequences; warps meet only where a (sequence, kv head) ends.
//  * The products run on mma.sync (m16n8k16, fp16): a chunk's keys are the 16 rows, the query rows the 8 columns, the G heads of the
//    group together.  A code is an fp16 number exactly; a query row is divided by a power of two so that its entries are at most 1.
//    Both scales stay in fp32: k_scale on the scores, v_scale on the weights, before they are rounded to fp16.
//  * The weights are kept relative to a maximum M of s_j + log2 v_scale[j] (not of s_j), so that the fp16 number w_j * v_scale[j] is at
//    most 2^8 and small scales lose nothing.  M moves only when a weight passes 2^8: the common chunk has one vote and no shuffles.
#include <math.h>

#include "mma_sync.cuh"
#include "rows8.cuh"

namespace llmi {

constexpr int RW8_WARPS = 8;
constexpr int RW8_MAX_ENTRIES = 4096;      // (sequence, row tile)s of a call
constexpr float RW8_LAZY = 256.f;          // weights up to this before the reference maximum moves
constexpr float RW8_TINY = 6.1629758e-33f; // 2^-107: no scale but 0 is smaller

struct Rows8Params {
  const __nv_bfloat16* q;
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
  int n_seqs, group, row_tiles;
  float scale_log2;
  int window;
  float* slots;                 // [2 * blocks][REGS][32]
  int* tickets;                 // [n_seqs * row_tiles * n_kv_heads], zero before and after
};

template <int D, int NT>
struct Rw8Cfg {
  static constexpr int KC = 2048 / D;              // keys of a chunk
  static constexpr int CPP = PAGE8 / KC;           // chunks of a page
  static constexpr int MT = KC / 16, KS = D / 16;  // key tiles of a chunk; 16-dim steps of a row
  static constexpr int STAGE = 4096 + 8 * KC;
  static constexpr int STAGES = 3;
  static constexpr int OREGS = KS * NT * 4, REGS = OREGS + 4 * NT;
  static constexpr int BLOCKS = REGS <= 44 ? 2 : 1;      // blocks a SM
  static constexpr int RING = RW8_WARPS * STAGES * STAGE;
  static constexpr int MERGE = 2 * REGS * 32 * 4;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Four codes as fp16 numbers: bytes 0, 1 and bytes 2, 3.
template <int HELD> __device__ __forceinline__ void halves4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (HELD == HELD_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    asm("prmt.b32 %0, %1, %2, 0x4140;" : "=r"(lo) : "r"(u), "r"(0x64646464u));
    asm("prmt.b32 %0, %1, %2, 0x4342;" : "=r"(hi) : "r"(u), "r"(0x64646464u));
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    lo = as_u32(__hsub2(*reinterpret_cast<__half2*>(&lo), bias));
    hi = as_u32(__hsub2(*reinterpret_cast<__half2*>(&hi), bias));
  } else {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  }
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }

// One (sequence, row tile): its rows and the pages that they see.
struct Rw8Entry {
  int seq, q_start, row0, rows, pos0, last, lo, pg_first, n_pages;
};
__device__ __forceinline__ Rw8Entry rw8_entry(const Rows8Params& p, int e, int tile_rows) {
  Rw8Entry d;
  d.seq = e / p.row_tiles;
  d.row0 = (e - d.seq * p.row_tiles) * tile_rows;
  d.q_start = p.seq_q_start[d.seq];
  const int q_len = p.seq_q_start[d.seq + 1] - d.q_start, kv_len = p.seq_kv_len[d.seq];
  d.rows = min(tile_rows, q_len * p.group - d.row0);
  d.pos0 = kv_len - q_len;
  d.n_pages = 0;
  if (d.rows <= 0 || kv_len <= 0) return d;
  const int first = d.pos0 + d.row0 / p.group;
  d.last = d.pos0 + (d.row0 + d.rows - 1) / p.group;
  d.lo = (p.window > 0 && first - p.window + 1 > 0) ? first - p.window + 1 : 0;
  d.pg_first = d.lo / PAGE8;
  if (d.last >= 0) d.n_pages = d.last / PAGE8 - d.pg_first + 1;
  return d;
}

template <int D, int NT, int HELD>
__global__ void __launch_bounds__(RW8_WARPS * 32, (Rw8Cfg<D, NT>::BLOCKS)) attention_rows8_kernel(Rows8Params p, int n_entries, int min_units) {
  using C = Rw8Cfg<D, NT>;
  constexpr int KC = C::KC, CPP = C::CPP, MT = C::MT, KS = C::KS, STAGES = C::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge_buf = reinterpret_cast<float*>(smem + C::RING);
  int* prefix = reinterpret_cast<int*>(smem + C::RING + C::MERGE);      // [n_entries + 1] pages ahead of an entry
  __shared__ int s_scan[RW8_WARPS], s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.group, Hkv = p.kv.n_kv_heads;
  pdl_wait();
  pdl_launch_dependents();

  // ---- the line of units: pages ahead of each entry ----
  {
    int carry = 0;
    for (int e0 = 0; e0 < n_entries; e0 += RW8_WARPS * 32) {
      const int e = e0 + threadIdx.x;
      const int n = e < n_entries ? rw8_entry(p, e, 8 * NT).n_pages : 0;
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_scan[warp] = x;
      __syncthreads();
      int before = carry, all = carry;
      for (int w = 0; w < RW8_WARPS; ++w) {
        if (w < warp) before += s_scan[w];
        all += s_scan[w];
      }
      if (e < n_entries) prefix[e] = before + x - n;
      carry = all;
      __syncthreads();
    }
    if (threadIdx.x == 0) prefix[n_entries] = carry;
    __syncthreads();
  }
  const int total = prefix[n_entries] * Hkv;
  const int blocks = max(1, min((int)gridDim.x, total / min_units));
  auto range_start = [&](int c) { return (int)((long)c * total / blocks); };
  if (blockIdx.x >= blocks || total == 0) return;
  const int u0 = range_start(blockIdx.x), u1 = range_start(blockIdx.x + 1);

  // ---- the ring: this warp's chunks of the block's range, asked for in order ----
  uint8_t* ring = smem + warp * STAGES * C::STAGE;
  struct Cursor {
    int unit, seg_end;       // the chunk's unit; where the units of its (entry, kv head) end
    int sub, e, kvh, pages, pg_first, seq;
  } in;
  auto find_entry = [&](int unit) {        // the entry whose units hold `unit`
    int a = 0, b = n_entries;              // prefix[a] * Hkv <= unit < prefix[b] * Hkv
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (prefix[m] * Hkv <= unit) a = m;
      else b = m;
    }
    return a;
  };
  auto seek = [&](Cursor& c) {             // the (entry, kv head) of c.unit
    c.e = find_entry(c.unit);
    const Rw8Entry d = rw8_entry(p, c.e, 8 * NT);
    c.pages = d.n_pages;
    c.pg_first = d.pg_first;
    c.seq = d.seq;
    c.kvh = (c.unit - prefix[c.e] * Hkv) / d.n_pages;
    c.seg_end = prefix[c.e] * Hkv + (c.kvh + 1) * d.n_pages;
  };
  in.unit = u0 + warp / CPP;
  in.sub = warp % CPP;
  static_assert(RW8_WARPS % CPP == 0, "a warp keeps its place in a page");
  int next_page = 0;
  auto look_up = [&]() {                   // the page of the chunk that is asked for next
    if (in.unit >= u1) return;
    if (in.unit >= in.seg_end) seek(in);
    const int i = in.pg_first + in.unit - (in.seg_end - in.pages);
    next_page = i < p.kv.table_pages ? p.kv.seq_pages[(size_t)in.seq * p.kv.pages_stride + i] : -1;
  };
  int issued = 0;
  auto issue = [&]() {
    if (in.unit < u1) {
      uint8_t* st = ring + (issued % STAGES) * C::STAGE;
      const bool known = (unsigned)next_page < (unsigned)p.kv.n_pages;
      const size_t row0 = ((size_t)(known ? next_page : 0) * Hkv + in.kvh) * PAGE8 + in.sub * KC;
      const uint8_t* kc = p.k_codes + row0 * D;
      const uint8_t* vc = p.v_codes + row0 * D;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        constexpr int UPR = D / 16;        // 16-byte pieces of a row
        const int x = lane + 32 * i, r = x / UPR, u = x % UPR;
        // Where a piece lies, so that no two lanes of a load meet in a bank.  Keys in the order of the rows of the product's tile
        // (key r is row 2 (r & 3) + (r >> 2 & 1) of its eight), pieces of odd rows of 128 bytes exchanged; values row by row.
        const int kr = (r & ~7) | ((r & 3) << 1) | ((r >> 2) & 1);
        const int ku = D == 128 ? u ^ ((kr & 1) << 2) : u;
        const int vu = D == 128 ? u ^ ((r & 3) << 1) : u ^ (((r >> 1) & 1) << 1);
        cp_async16(st + kr * D + ku * 16, kc + x * 16, 16);
        cp_async16(st + 2048 + r * D + vu * 16, vc + x * 16, 16);
      }
      if (known) {
        if (lane < KC / 4) cp_async16(st + 4096 + lane * 16, p.k_scales + row0 + lane * 4, 16);
        else if (lane < KC / 2) cp_async16(st + 4096 + lane * 16, p.v_scales + row0 + (lane - KC / 4) * 4, 16);
      } else {                             // a page that the pool does not have reads as NaN
        for (int i = lane; i < 2 * KC; i += 32) reinterpret_cast<float*>(st + 4096)[i] = __int_as_float(0x7fffffff);
      }
      in.unit += RW8_WARPS / CPP;
      look_up();
    }
    cp_async_commit();
    ++issued;
  };
  in.seg_end = 0;
  look_up();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue();

  float O[KS][NT][4], M[NT][2], L[NT][2];
  // lanes' registers <-> 32 consecutive floats a register: the state of a (range, entry, kv head)
  auto put = [&](float* at) {
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) at[((i * NT + n) * 4 + j) * 32 + lane] = O[i][n][j];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        at[(C::OREGS + 2 * n + j) * 32 + lane] = M[n][j];
        at[(C::OREGS + 2 * NT + 2 * n + j) * 32 + lane] = L[n][j];
      }
  };
  // this state and another one, each relative to its own maximum (a state without one is zeros, or NaN, as it is)
  auto join = [&](auto value) {
    float mine[NT][2], other[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float mo = value(C::OREGS + 2 * n + j), m = fmaxf(M[n][j], mo);
        mine[n][j] = M[n][j] == -INFINITY ? 1.f : fast_exp2(M[n][j] - m);
        other[n][j] = mo == -INFINITY ? 1.f : fast_exp2(mo - m);
        M[n][j] = m;
        L[n][j] = L[n][j] * mine[n][j] + value(C::OREGS + 2 * NT + 2 * n + j) * other[n][j];
      }
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) O[i][n][j] = O[i][n][j] * mine[n][j & 1] + value((i * NT + n) * 4 + j) * other[n][j & 1];
  };
  auto clear = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) M[n][j] = -INFINITY, L[n][j] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) O[i][n][j] = 0.f;
    }
  };
  // the eight warps' states into warp 0's, two at a time
  auto join_warps = [&]() {
#pragma unroll
    for (int from = RW8_WARPS - 2; from >= 0; from -= 2) {
      const int n = from == 0 ? 1 : 2, to = from == 0 ? 0 : from - 2;      // warps from .. to warps to .. (last: warp 1 to warp 0)
      const int first = from == 0 ? 1 : from;
      if (warp >= first && warp < first + n) put(merge_buf + (warp - first) * C::REGS * 32);
      __syncthreads();
      if (warp >= to && warp < to + n) {
        const float* at = merge_buf + (warp - to) * C::REGS * 32 + lane;
        join([&](int i) { return at[i * 32]; });
      }
      __syncthreads();
    }
  };

  // ---- segments: the block's part of one (entry, kv head) after the other ----
  int taken = 0;                           // chunks that this warp has worked through
  int unit = u0 + warp / CPP;              // and its next one's unit
  const int key_sub = (warp % CPP) * KC;
  for (int seg = u0; seg < u1;) {
    const int e = find_entry(seg);
    const Rw8Entry d = rw8_entry(p, e, 8 * NT);
    const int kvh = (seg - prefix[e] * Hkv) / d.n_pages;
    const int begin = prefix[e] * Hkv + kvh * d.n_pages, end = begin + d.n_pages;
    const int seg_end = min(end, u1);

    // queries: row n * 8 + g, its dims in the order in which a lane has the keys' codes
    uint32_t qf[NT][KS][2];
    float fac[NT][2];                      // of the columns 2t, 2t + 1: scale * log2(e) * the row's power of two
    int col_pos[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = n * 8 + g;
      float x[D / 4];
      float a = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 raw = make_uint4(0u, 0u, 0u, 0u);
          if (r < d.rows) {
            const int row = d.row0 + r;
            raw = *reinterpret_cast<const uint4*>(p.q + (size_t)(d.q_start + row / G) * p.ldq + (size_t)(kvh * G + row % G) * D + 64 * c + 16 * t + 8 * h);
          }
          const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(b[i]);
            x[c * 16 + h * 8 + 2 * i] = f.x;
            x[c * 16 + h * 8 + 2 * i + 1] = f.y;
            a = fmaxf(a, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
      a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
      a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
      // the power of two above the row's largest entry (a row that is zero or not finite: 1)
      int ex = 0;
      if (a > 0.f && a <= FLT_MAX) ex = max(-100, (int)((__float_as_uint(a) >> 23) & 255) - 126);
      const float down = __uint_as_float((uint32_t)(127 - min(ex, 126)) << 23), down2 = ex > 126 ? 1.f / (float)(1 << (ex - 126)) : 1.f;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) qf[n][s][h] = pack_half2(x[4 * s + 2 * h] * down * down2, x[4 * s + 2 * h + 1] * down * down2);
      const float f = ldexpf(p.scale_log2, ex);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        fac[n][j] = __shfl_sync(0xffffffffu, f, (2 * t + j) * 4);
        const int r2 = n * 8 + 2 * t + j;
        col_pos[n][j] = d.pos0 + (d.row0 + min(r2, d.rows - 1)) / G;
      }
    }
    const int first_pos = d.pos0 + d.row0 / G;
    clear();
    bool unset = true;                     // some column has no maximum yet
    for (; unit < seg_end; unit += RW8_WARPS / CPP) {
      cp_async_wait<STAGES - 2>();
      __syncwarp();                        // every lane's copies are here, and every lane is done with the stage before
      issue();
      const uint8_t* st = ring + (taken % STAGES) * C::STAGE;
      const float* ks_s = reinterpret_cast<const float*>(st + 4096);
      const float* vs_s = ks_s + KC;
      const int key0 = (d.pg_first + unit - begin) * PAGE8 + key_sub;
      const bool masked = key0 + KC - 1 > first_pos || (p.window > 0 && key0 <= d.last - p.window);
      float x[MT][NT][4], vs[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t ka[KS], kb[KS];
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const int u = D == 128 ? ((4 * c + t) ^ ((g & 1) << 2)) : t;
          const uint4 va = *reinterpret_cast<const uint4*>(st + (m * 16 + g) * D + u * 16);
          const uint4 vb = *reinterpret_cast<const uint4*>(st + (m * 16 + 8 + g) * D + u * 16);
          ka[4 * c] = va.x, ka[4 * c + 1] = va.y, ka[4 * c + 2] = va.z, ka[4 * c + 3] = va.w;
          kb[4 * c] = vb.x, kb[4 * c + 1] = vb.y, kb[4 * c + 2] = vb.z, kb[4 * c + 3] = vb.w;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) x[m][n][j] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          uint32_t a[4];
          halves4<HELD>(ka[s], a[0], a[2]);
          halves4<HELD>(kb[s], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(x[m][n], a, qf[n][s][0], qf[n][s][1]);
        }
        // rows g and g + 8 of the tile are the keys pk and pk + 8
        const int pk = m * 16 + (g >> 1) + 4 * (g & 1);
        const float ks0 = ks_s[pk], ks1 = ks_s[pk + 8];
        vs[m][0] = vs_s[pk], vs[m][1] = vs_s[pk + 8];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[m][n][j] *= (j < 2 ? ks0 : ks1) * fac[n][j & 1];
            if (masked) {
              const int key = key0 + pk + (j < 2 ? 0 : 8);
              if (key > col_pos[n][j & 1] || (p.window > 0 && key <= col_pos[n][j & 1] - p.window)) x[m][n][j] = -INFINITY;
            }
          }
      }
      float ex[MT][NT][4];
      auto weigh = [&]() {                 // -> the largest weight times value scale
        float top = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float neg = M[n][j & 1] == -INFINITY ? 0.f : -M[n][j & 1];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              ex[m][n][j] = fast_exp2(x[m][n][j] + neg);
              top = fmaxf(top, ex[m][n][j] * fmaxf(vs[m][j >> 1], RW8_TINY));
            }
          }
        return top;
      };
      float top = unset ? INFINITY : weigh();
      if (__any_sync(0xffffffffu, top > RW8_LAZY)) {
        unset = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = -INFINITY;
#pragma unroll
            for (int m = 0; m < MT; ++m)
              mx = fmaxf(mx, fmaxf(x[m][n][j] + fast_log2(fmaxf(vs[m][0], RW8_TINY)), x[m][n][j + 2] + fast_log2(fmaxf(vs[m][1], RW8_TINY))));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(M[n][j], mx), f = M[n][j] == -INFINITY ? 1.f : fast_exp2(M[n][j] - m_new);
            L[n][j] *= f;
#pragma unroll
            for (int i = 0; i < KS; ++i) O[i][n][j] *= f, O[i][n][j + 2] *= f;
            M[n][j] = m_new;
            unset = unset || m_new == -INFINITY;
          }
        unset = __any_sync(0xffffffffu, unset);
        weigh();
      }
      const int seen0 = max(d.lo - key0, 0), seen1 = d.last - key0;      // rows of the chunk that some query sees
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            L[n][j & 1] += ex[m][n][j];
            w[j] = ex[m][n][j] * vs[m][j >> 1];
            if (masked && x[m][n][j] == -INFINITY) w[j] = 0.f;           // (its scale may be anything)
          }
          pb[n][0] = transpose8x8(pack_half2(w[0], w[1]));
          pb[n][1] = transpose8x8(pack_half2(w[2], w[3]));
        }
        // values: keys 2t, 2t + 1 (+ 8) of the tile are the rows t, t + 4 (+ 8); a lane has the dims g * D / 8 ..
        uint32_t vw[4][D / 32];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = m * 16 + t + 4 * (j & 1) + 8 * (j >> 1);
          if (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(st + 2048 + r * D + ((g ^ ((r & 3) << 1)) * 16));
            vw[j][0] = v.x, vw[j][1] = v.y, vw[j][D / 32 - 2] = v.z, vw[j][D / 32 - 1] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(st + 2048 + r * D + (((g >> 1) ^ (((r >> 1) & 1) << 1)) * 16) + (g & 1) * 8);
            vw[j][0] = v.x, vw[j][1] = v.y;
          }
          if (masked && (r < seen0 || r > seen1)) {                      // (what lies there may be no number)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) vw[j][i] = 0u;
          }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {       // four dims: two tiles of dims
          uint32_t z[4], a01[4], a23[4];
          asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(z[0]) : "r"(vw[0][w]), "r"(vw[1][w]));
          asm("prmt.b32 %0, %1, %2, 0x7362;" : "=r"(z[1]) : "r"(vw[0][w]), "r"(vw[1][w]));
          asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(z[2]) : "r"(vw[2][w]), "r"(vw[3][w]));
          asm("prmt.b32 %0, %1, %2, 0x7362;" : "=r"(z[3]) : "r"(vw[2][w]), "r"(vw[3][w]));
          halves4<HELD>(z[0], a01[0], a01[1]);
          halves4<HELD>(z[2], a01[2], a01[3]);
          halves4<HELD>(z[1], a23[0], a23[1]);
          halves4<HELD>(z[3], a23[2], a23[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(O[2 * w][n], a01, pb[n][0], pb[n][1]);
            mma_f16(O[2 * w + 1][n], a23, pb[n][0], pb[n][1]);
          }
        }
      }
      ++taken;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) L[n][j] += __shfl_xor_sync(0xffffffffu, L[n][j], o);
    join_warps();
    bool whole = true;
    if (begin < u0 || end > u1) {          // other blocks have units of it too
      auto block_of = [&](int u) {         // the block whose range holds unit u
        int c = (int)((long)u * blocks / total);
        while (range_start(c + 1) <= u) ++c;
        while (range_start(c) > u) --c;
        return c;
      };
      const int c_first = block_of(begin), c_last = block_of(end - 1);
      auto slot = [&](int c) { return p.slots + (size_t)(2 * c + (range_start(c) < begin ? 1 : 0)) * C::REGS * 32; };
      int* ticket = p.tickets + (size_t)e * Hkv + kvh;
      if (warp == 0) {
        put(slot(blockIdx.x));
        __threadfence();
        __syncwarp();
        if (lane == 0) s_last = atomicAdd(ticket, 1) == c_last - c_first;
      }
      __syncthreads();
      whole = s_last != 0;
      if (whole) {
        __threadfence();
        clear();
        for (int c = c_first + warp; c <= c_last; c += RW8_WARPS) {
          const float* at = slot(c) + lane;
          join([&](int i) { return __ldcg(at + i * 32); });
        }
        join_warps();
        if (threadIdx.x == 0) *ticket = 0;
      }
      __syncthreads();                     // (s_last is free again)
    }
    if (whole && warp == 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int r = n * 8 + 2 * t + j;
          if (r >= d.rows) continue;
          const int row = d.row0 + r;
          const float inv = L[n][j] == 0.f ? 0.f : 1.f / L[n][j];
          __nv_bfloat16* o = p.out + (size_t)(d.q_start + row / G) * p.ldo + (size_t)(kvh * G + row % G) * D + g * (D / 8);
#pragma unroll
          for (int w = 0; w < D / 64; ++w) {     // eight dims
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              __nv_bfloat162 h = __floats2bfloat162_rn(O[4 * w + i][n][j] * inv, O[4 * w + i][n][j + 2] * inv);
              v[i] = *reinterpret_cast<uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(o + 8 * w) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
    }
    seg = seg_end;
  }
  cp_async_wait_all();
}

template <int D, int NT, int HELD> bool rw8_configured() {
  static PerDevice<bool> done;
  if (!done.here())
    done.here() = cudaFuncSetAttribute(attention_rows8_kernel<D, NT, HELD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Rw8Cfg<D, NT>::RING + Rw8Cfg<D, NT>::MERGE + 4 * (RW8_MAX_ENTRIES + 1)) == cudaSuccess;
  return done.here();
}

template <int D, int NT, int HELD> int launch_rows8(const Rows8Params& p, int n_entries, int grid, cudaStream_t stream) {
  using C = Rw8Cfg<D, NT>;
  if (!rw8_configured<D, NT, HELD>()) return LLMI_ERR_LAUNCH;
  const size_t smem = C::RING + C::MERGE + 4 * ((size_t)n_entries + 1);
  // no more blocks than are resident: many entries' table may leave room for one a SM only (228 KB; a block's own 1 KB and its statics)
  const int fit = (int)((228 << 10) / (smem + 1280));
  const int resident = min(C::BLOCKS, max(1, fit)) * sm_count();
  return launch_pdl(PDL_ATTENTION, attention_rows8_kernel<D, NT, HELD>, (unsigned)min(grid, resident), RW8_WARPS * 32, smem, stream, p, n_entries, RW8_WARPS / C::CPP);
}

// query rows of a tile, in eighths: the fewest that hold a sequence's rows, of those there are
inline int rw8_tiles(int D, long rows) { return rows <= 8 ? 1 : (rows <= 16 || D == 128) ? 2 : 4; }
inline int rw8_regs(int D, int nt) { return D / 16 * nt * 4 + 4 * nt; }
inline int rw8_grid(int D, int nt, long units) {
  const long n = (long)(rw8_regs(D, nt) <= 44 ? 2 : 1) * sm_count();
  return (int)(units < n ? units : n);
}

}  // namespace llmi

using namespace llmi;

// What a call needs: *floats of scratch for the blocks' partial results, *ints tickets (zero before the first call; every call
// leaves them zero).  `max_q`: most tokens that a sequence brings.
LLMI_EXPORT int llmi_attention_rows8_workspace(int n_seqs, int max_q, int n_heads, int n_kv_heads, int head_dim, int table_pages, long* floats, long* ints) {
  if (n_seqs <= 0 || max_q <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || (head_dim != 64 && head_dim != 128) || table_pages <= 0) return LLMI_ERR_BAD_SIZE;
  const long rows = (long)max_q * (n_heads / n_kv_heads);
  const int nt = rw8_tiles(head_dim, rows);
  const long tiles = (rows + 8 * nt - 1) / (8 * nt);
  if (n_seqs * tiles > RW8_MAX_ENTRIES || n_seqs * tiles * n_kv_heads * (long)table_pages > 0x7fffffffL) return LLMI_ERR_BAD_SIZE;
  *ints = n_seqs * tiles * n_kv_heads;
  *floats = 2L * rw8_grid(head_dim, nt, n_seqs * tiles * n_kv_heads * (long)table_pages) * rw8_regs(head_dim, nt) * 32;
  return LLMI_OK;
}

LLMI_EXPORT int llmi_attention_rows8(int held, const void* q, long ldq, void* out, long ldo, const void* k_codes, const float* k_scales,
                                     const void* v_codes, const float* v_scales, const int32_t* seq_q_start, const int32_t* seq_kv_len,
                                     const int32_t* seq_pages, int pages_stride, int table_pages, int n_seqs, int n_pages, int max_q,
                                     int n_heads, int n_kv_heads, int head_dim, float scale, int window, float* slots, long n_floats, int* tickets,
                                     long n_ints, cudaStream_t stream) {
  long floats, ints;
  const int rc = llmi_attention_rows8_workspace(n_seqs, max_q, n_heads, n_kv_heads, head_dim, table_pages, &floats, &ints);
  if (rc != LLMI_OK) return rc;
  if (n_floats < floats || n_ints < ints || n_pages <= 0 || window < 0) return LLMI_ERR_BAD_SIZE;
  if (held != HELD_INT8 && held != HELD_E4M3) return LLMI_ERR_BAD_DTYPE;
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales) & 15) || (ldq & 7) || (ldo & 7))
    return LLMI_ERR_ALIGN;
  const int group = n_heads / n_kv_heads;
  const long rows = (long)max_q * group;
  const int nt = rw8_tiles(head_dim, rows), tiles = (int)((rows + 8 * nt - 1) / (8 * nt));
  Rows8Params p{(const __nv_bfloat16*)q, ldq, (__nv_bfloat16*)out, ldo, (const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales,
                seq_q_start, seq_kv_len, Paged8{seq_pages, pages_stride, table_pages, n_pages, n_kv_heads, head_dim}, n_seqs, group, tiles,
                scale * 1.4426950408889634f, window, slots, tickets};
  const int n_entries = n_seqs * tiles, grid = rw8_grid(head_dim, nt, (long)n_entries * n_kv_heads * table_pages);
#define LLMI_ROWS8(D_, NT_) \
  (held == HELD_INT8 ? launch_rows8<D_, NT_, HELD_INT8>(p, n_entries, grid, stream) : launch_rows8<D_, NT_, HELD_E4M3>(p, n_entries, grid, stream))
  if (head_dim == 64) return nt == 1 ? LLMI_ROWS8(64, 1) : nt == 2 ? LLMI_ROWS8(64, 2) : LLMI_ROWS8(64, 4);
  return nt == 1 ? LLMI_ROWS8(128, 1) : LLMI_ROWS8(128, 2);
#undef LLMI_ROWS8
}
