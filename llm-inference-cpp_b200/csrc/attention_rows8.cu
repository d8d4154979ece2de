// Attention of few query rows a sequence — single tokens, short messages — over the paged cache held in 8 bits (rows8.cuh), head
// size 64 or 128.  For a row at position p of kv head g, over the keys j of its sequence it sees:
//     s_j = scale * k_scale[j] * (q . k_code[j]),   w = softmax(s),   out = sum_j w_j * v_scale[j] * v_code[j]
// (reference loop: src/model/transformer.cpp:263-282).  Every code is read once and takes part in a handful of operations, so what
// bounds the kernel is HBM: 2 (D + 4) bytes a position and kv head; behind that the instructions that make codes fp16 numbers, and
// the join.  Measured: 8 x 4,096 positions of 32 heads of 64 30 us with the append (4.7 TB/s), 60,001 to 131,071 positions of three
// sequences 41 us (4.5), 64 of 200 to 4,400, 32 heads by 8 of 128, 46 us (4.0); a copy reaches 6.5.
//
//  * All pages that the step's rows see, kv head by kv head and sequence by sequence, are one line of units (a unit: one page of one
//    kv head), cut into as many equal ranges as there are blocks resident on the device.  A block works through its range whatever
//    the sequences' lengths are, so no block waits for the longest one, and nothing about the cut depends on what the host knows.
//    A (sequence, kv head) that several ranges share leaves partial results, which a second kernel adds in the order of the ranges:
//    the same call gives the same bits.  (Joined by the block that draws the last of a pair's tickets it took 12 to 17 us behind 22 to
//    28 us of streaming: fences, atomics and cold code, one behind the other.)  Where there are no more of them than resident blocks
//    and they are of about one length, or short, each has a block of its own instead.
//  * Within a block each warp takes every eighth chunk (2 KB of key codes, 2 KB of value codes, their scales) into a ring of its own
//    in shared memory with cp.async, across the borders of sequences; warps meet only where a (sequence, kv head) ends, through the
//    stages that they have just read.
//  * The products run on mma.sync (m16n8k16, fp16): a chunk's keys are the 16 rows, the query rows the 8 columns, the G heads of the
//    group together.  A code is an fp16 number exactly; a query row is multiplied by a power of two that brings its largest entry near
//    2^15, so that smaller ones keep their bits as far down as fp16 reaches: a bf16 query is exact down to 2^-29 of the largest, the
//    32-bit ones that `rope` makes of bf16 rows are rounded to 11 bits.
//    Both scales stay in fp32: k_scale on the scores, v_scale on the weights, before they are rounded to fp16.  In the 32-bit path
//    queries and weights are the sums of two fp16 numbers (22 bits), the second of a weight 2^11 as large as it counts, so that small
//    weights have it too; sixteen keys' sum is added to the output's in fp32, and the weights' sum is compensated (Kahan).
//  * The weights are kept relative to a maximum M of s_j + log2 v_scale[j] (not of s_j), so that small scales lose nothing: the fp16
//    number w_j * v_scale[j] is 2^7 for the largest when M moves, and M moves only when one passes 2^15 — the common chunk has one vote
//    and no shuffles.  A weight keeps 11 bits down to 2^-21 of the row's largest; below that it is off by at most 2^-32 of the largest
//    (32-bit path: 22 bits, 2^-43).  Many small weights beside a large one need them that far down: of 32,000 keys 17.5 nats below
//    another an eighth, its warp's, was lost with M 2^7 higher: 1e-4 of the output.
#include <math.h>

#include <type_traits>

#include "mma_sync.cuh"
#include "rows8.cuh"

namespace llmi {

constexpr int RW8_WARPS = 8;
constexpr int RW8_MAX_ENTRIES = 4096;      // (sequence, row tile)s of a call, and sequences
constexpr float RW8_UP = 7.f;              // the largest weight is 2^7 where the reference maximum has moved
constexpr float RW8_LAZY = 32768.f;        // weights up to 2^15 before it moves
constexpr float RW8_SUM = 5.192296858534828e33f;   // 2^112: a sum of weights up to this (keys whose values are zeros may weigh that much)
constexpr float RW8_TINY = 1.0097419586828951e-28f; // 2^-93: smaller value scales count as this where M is made

struct Rows8Params {
  const void* q;
  long ldq;
  void* out;
  long ldo;
  const uint8_t* k_codes;
  const float* k_scales;
  const uint8_t* v_codes;
  const float* v_scales;
  const int32_t* seq_q_start;   // [n_seqs + 1]
  const int32_t* seq_kv_len;    // [n_seqs]
  Paged8 kv;
  int n_seqs, group;
  int row_tiles;                // most row tiles of a sequence
  float scale_log2;
  int window;
  int q_f32;                    // q is fp32 (where out is bf16)
  float* slots;                 // [2 * blocks][SLOT]: partial results, of a block's first segment and of its last
  int* whose;                   // [2 * blocks]: 0, or (its (sequence, row tile, kv head) + 1) * 2 + whether it is the first of the parts
};

// D: head size; NT: eighths of query rows; T: the type of q and out (float: two fp16 numbers each).
template <int D, int NT, typename T>
struct Rw8Cfg {
  static constexpr int SP = std::is_same<T, float>::value ? 2 : 1;
  static constexpr bool SEVERAL = NT == (SP == 2 ? 2 : 4) * 64 / D;      // a sequence may have several row tiles: rw8_tiles' widest
  static constexpr int KC = D == 64 && NT == 1 ? 32 : 16;          // keys of a chunk
  static constexpr int CPP = PAGE8 / KC;           // chunks of a page
  static constexpr int MT = KC / 16, KS = D / 16;  // key tiles of a chunk; 16-dim steps of a row
  static constexpr int CODES = KC * D;             // bytes of a chunk's key codes, and of its value codes
  static constexpr int STAGE = 2 * CODES + 8 * KC;
  static constexpr int PAIRS = KS * NT;            // tiles of 16 dims by 8 rows of an output
  static constexpr int STATE = (PAIRS * 4 * 32 + 16 * NT) * 4;      // bytes of a state: outputs, then maxima and sums of the rows
  static constexpr bool IN_RING = STATE <= STAGE;  // a warp's state fits the stage it has just read
  static constexpr int BLOCKS = (SP == 1 && PAIRS <= 8) ? 2 : 1;    // blocks a SM
  static constexpr int STAGES = STAGE < 4000 ? (BLOCKS == 2 ? 4 : 6) : (BLOCKS == 2 ? 3 : 4);
  static constexpr int RING = RW8_WARPS * STAGES * STAGE;
  static constexpr int MERGE = IN_RING ? 0 : RW8_WARPS * STATE;
  static constexpr int SLOT = STATE / 4;           // floats of a block's partial result
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) { return as_u32(__floats2half2_rn(lo, hi)); }

// How the line of units is cut.  In pages: what a (sequence, kv head) costs beside its pages (its queries, the join of the warps, its
// output), as units of no page at the front of its own; the most pages of the longest where each has a block of its own whatever their
// number (the join of parts is a kernel of 4 us, 8 pages' time); the least a range has (one query head row, 9 heads of 64 by 3, 2,000
// positions: 12.0 us in ranges of 16, 9.4 of 8, 9.0 of 4; 32 heads of 128 by 8, 4,000: 15.0 of 8, 16.3 of 4, 19.7 of 2: a part costs the
// join as well); how near a border of two (sequence, kv head)s a cut is moved to it.
struct Rw8Cut {
  int front, most_whole, least, near;
};

// One (sequence, row tile), number sequence * row_tiles + tile: its rows and the pages that they see.
struct Rw8Entry {
  int seq, q_start, row0, rows, pos0, last, lo, pg_first, n_pages;
};
__device__ __forceinline__ Rw8Entry rw8_entry(const Rows8Params& p, int number, int tile_rows) {
  Rw8Entry d;
  d.seq = number / p.row_tiles;
  d.row0 = (number - d.seq * p.row_tiles) * tile_rows;
  d.q_start = p.seq_q_start[d.seq];
  const int q_len = p.seq_q_start[d.seq + 1] - d.q_start, kv_len = p.seq_kv_len[d.seq];
  d.rows = min(tile_rows, q_len * p.group - d.row0);
  d.pos0 = kv_len - q_len;
  d.n_pages = 0;
  if (d.rows <= 0 || kv_len <= 0) return d;
  const int first = d.pos0 + d.row0 / p.group;
  d.last = d.pos0 + (d.row0 + d.rows - 1) / p.group;
  d.lo = (p.window > 0 && first - p.window + 1 > 0) ? first - p.window + 1 : 0;
  d.pg_first = page_index8(p.kv, d.lo);
  if (d.last >= 0) d.n_pages = page_index8(p.kv, d.last) - d.pg_first + 1;
  return d;
}

// One tile of an output — 16 dims by 8 rows — out of several states (a state without a maximum is zeros, or NaN, as it is), eight at a time.
struct Rw8Tile {
  float o[4], m[2], l[2];
};
template <typename C, int NT, typename State, typename Load>
__device__ __forceinline__ Rw8Tile rw8_gather(int pair, int first, int n_states, int step, State state, Load load) {
  const int lane = threadIdx.x & 31, n = pair % NT, t = lane & 3;
  Rw8Tile r;
  r.m[0] = r.m[1] = -INFINITY;
  r.l[0] = r.l[1] = r.o[0] = r.o[1] = r.o[2] = r.o[3] = 0.f;
  for (int w0 = first; w0 < n_states; w0 += 8 * step) {
    Rw8Tile x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* at = state(min(w0 + i * step, n_states - 1));
      const float* m = at + C::PAIRS * 128 + n * 8 + 2 * t;
#pragma unroll
      for (int j = 0; j < 2; ++j) x[i].m[j] = load(m + j), x[i].l[j] = load(m + 8 * NT + j);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i].o[j] = load(at + (pair * 4 + j) * 32 + lane);
    }
    float f[2], top[2] = {r.m[0], r.m[1]};
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) top[j] = fmaxf(top[j], x[i].m[j]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float down = r.m[j] == -INFINITY ? 0.f : r.m[j] - top[j];
      f[j] = fast_exp2(down), r.l[j] = rescale8(r.l[j], down), r.m[j] = top[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) r.o[j] *= f[j & 1];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (w0 + i * step >= n_states) break;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float down = x[i].m[j] == -INFINITY ? 0.f : x[i].m[j] - top[j];
        f[j] = fast_exp2(down), r.l[j] += rescale8(x[i].l[j], down);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) r.o[j] = fmaf(x[i].o[j], f[j & 1], r.o[j]);
    }
  }
  return r;
}
template <int D, int NT, typename T>
__device__ __forceinline__ void rw8_write(const Rows8Params& p, const Rw8Entry& d, int kvh, int pair, const Rw8Tile& r) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, G = p.group;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r8 = (pair % NT) * 8 + 2 * t + j;
    if (r8 >= d.rows) continue;
    const int row = d.row0 + r8;
    // (a position below 0 sees nothing: zeros; scores that are all -infinity: NaN)
    const float inv = d.pos0 + row / G < 0 ? 0.f : 1.f / r.l[j];
    T* at = (T*)p.out + (size_t)(d.q_start + row / G) * p.ldo + (size_t)(kvh * G + row % G) * D + g * (D / 8) + 2 * (pair / NT);
    if (sizeof(T) == 4) *reinterpret_cast<float2*>(at) = make_float2(r.o[j] * inv, r.o[j + 2] * inv);
    else *reinterpret_cast<__nv_bfloat162*>(at) = __floats2bfloat162_rn(r.o[j] * inv, r.o[j + 2] * inv);
  }
}

template <int D, int NT, int HELD, typename T>
__global__ void __launch_bounds__(RW8_WARPS * 32, (Rw8Cfg<D, NT, T>::BLOCKS)) attention_rows8_kernel(Rows8Params p, int n_entries, Rw8Cut cut) {
  using C = Rw8Cfg<D, NT, T>;
  constexpr int KC = C::KC, CPP = C::CPP, MT = C::MT, KS = C::KS, STAGES = C::STAGES, SP = C::SP, STEP = RW8_WARPS / C::CPP;
  static_assert(RW8_WARPS % CPP == 0, "a warp keeps its place in a page");
  extern __shared__ __align__(128) uint8_t smem[];
  int* prefix = reinterpret_cast<int*>(smem + C::RING + C::MERGE);      // [n_entries + 1] units ahead of an entry
  __shared__ int s_scan[RW8_WARPS], s_top[RW8_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = p.group, Hkv = p.kv.n_kv_heads;
  pdl_launch_dependents();
  // (ahead of the wait: the step's index block only, and the page table in it)

  // ---- entries: where a sequence may have several row tiles, those that there are, one sequence behind the other (how many each has is
  // known here only); else a sequence each.  The line of units: units ahead of each entry ----
  uint16_t* starts = reinterpret_cast<uint16_t*>(prefix + n_entries + 1);      // [n_seqs + 1] tiles ahead of a sequence (where row_tiles > 1)
  auto last_before = [](const auto* ahead, int n, int x) {      // the i with ahead[i] <= x < ahead[i + 1] (the last one if x is behind all)
    int a = 0, b = n;
    while (b - a > 1) {
      const int m = (a + b) >> 1;
      if (ahead[m] <= x) a = m;
      else b = m;
    }
    return a;
  };
  auto number_of = [&](int e) {            // of an entry, as rw8_entry takes it (-1: there are fewer)
    if (!C::SEVERAL || p.row_tiles == 1) return e;
    if (e >= starts[p.n_seqs]) return -1;
    const int seq = last_before(starts, p.n_seqs, e);
    return seq * p.row_tiles + e - starts[seq];
  };
  int pairs = 0, longest = 0;              // (entry, kv head)s that have pages; the most pages of one
  auto line_up = [&](auto* into, int count, auto of) {          // into[i] = the sum of `of` (number, pages) over all ahead of i
    constexpr int MOST = sizeof(*into) == 2 ? 0xffff : 0x7fffffff;
    int carry = 0;
    for (int i0 = 0; i0 < count; i0 += RW8_WARPS * 32) {
      const int i = i0 + threadIdx.x;
      const int2 mine = i < count ? of(i) : make_int2(0, 0);
      int x = mine.x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      const int top = __reduce_max_sync(0xffffffffu, mine.y);
      if (lane == 31) s_scan[warp] = x, s_top[warp] = top;
      pairs += __syncthreads_count(mine.y > 0) * Hkv;
      int before = carry, all = carry;
#pragma unroll
      for (int w = 0; w < RW8_WARPS; ++w) {
        if (w < warp) before += s_scan[w];
        all += s_scan[w];
        longest = max(longest, s_top[w]);
      }
      if (i < count) into[i] = min(before + x - mine.x, MOST);
      carry = all;
      __syncthreads();
    }
    if (threadIdx.x == 0) into[count] = min(carry, MOST);
    __syncthreads();
  };
  if (C::SEVERAL && p.row_tiles > 1)
    line_up(starts, p.n_seqs, [&](int seq) {
      const int rows = (p.seq_q_start[seq + 1] - p.seq_q_start[seq]) * G;
      return make_int2(p.seq_kv_len[seq] > 0 && rows > 0 ? min((rows + 8 * NT - 1) / (8 * NT), p.row_tiles) : 0, 0);
    });
  line_up(prefix, n_entries, [&](int e) {
    const int number = number_of(e), pages = number < 0 ? 0 : rw8_entry(p, number, 8 * NT).n_pages;
    return make_int2(pages > 0 ? (pages + cut.front) * Hkv : 0, pages);
  });
  const int total = prefix[n_entries];
  // each its own block, or the line in even ranges
  const bool whole = pairs <= (int)gridDim.x && (longest <= cut.most_whole || (5 * pairs >= 3 * (int)gridDim.x && (long)(longest + cut.front) * pairs <= total + total / 4));
  const int blocks = whole ? pairs : min((int)gridDim.x, max(total / cut.least, pairs));
  if (blockIdx.x >= blocks || total == 0) {
    pdl_wait();
    if (threadIdx.x < 2) p.whose[2 * blockIdx.x + threadIdx.x] = 0;
    return;
  }
  const int per = total / blocks, longer = total - per * blocks;      // even ranges: the first `longer` have per + 1 units
  auto find_entry = [&](int unit) { return last_before(prefix, n_entries, unit); };
  const int near = min(cut.near, per / 2);
  auto range_start = [&](int c) {          // an even cut, moved to the border of two (entry, kv head)s that is near
    const int u = c * per + min(c, longer);
    if (u >= total) return total;
    const int e = find_entry(u), len = (prefix[e + 1] - prefix[e]) / Hkv, at = (u - prefix[e]) % len;
    return at <= near ? u - at : len - at <= near ? u - at + len : u;
  };
  int u0, u1, e_first;
  if (whole) {
    // (its entry: the last one with no more than so many pairs ahead, found as the line's share of pairs: entries without pages take none)
    int rank = blockIdx.x / Hkv;
    e_first = -1;
    for (int e0 = 0; e_first < 0; e0 += 32) {
      const uint32_t some = __ballot_sync(0xffffffffu, e0 + lane < n_entries && prefix[e0 + lane + 1] > prefix[e0 + lane]);
      if (rank < __popc(some)) e_first = e0 + __fns(some, 0, rank + 1);
      else rank -= __popc(some);
    }
    const int len = (prefix[e_first + 1] - prefix[e_first]) / Hkv;
    u0 = prefix[e_first] + (blockIdx.x % Hkv) * len;
    u1 = u0 + len;
  } else {
    u0 = range_start(blockIdx.x), u1 = range_start(blockIdx.x + 1);
    e_first = find_entry(u0 < total ? u0 : 0);
  }
  if (u0 >= u1) {
    pdl_wait();
    if (threadIdx.x < 2) p.whose[2 * blockIdx.x + threadIdx.x] = 0;
    return;
  }
  // the block's part of the (entry, kv head) that has unit `at`, from there on
  struct Segment {
    Rw8Entry d;
    int number, kvh, begin, end;           // all units of the (entry, kv head)
    int first, n;                          // of its pages: the block's first, and how many
  };
  auto segment_at = [&](int at, int& e) {
    while (prefix[e + 1] <= at) ++e;
    Segment s;
    s.number = number_of(e);
    s.d = rw8_entry(p, s.number, 8 * NT);
    const int len = s.d.n_pages + cut.front;
    s.kvh = (at - prefix[e]) / len;
    s.begin = prefix[e] + s.kvh * len;
    s.end = s.begin + len;
    s.first = max(at - s.begin - cut.front, 0);
    s.n = max(min(s.end, u1) - s.begin - cut.front, 0) - s.first;
    return s;
  };

  // ---- the ring: this warp's chunks of the block's pages, asked for in order ----
  uint8_t* ring = smem + warp * STAGES * C::STAGE;
  const int sub = warp % CPP;              // the warp's place in a page
  struct {
    int page, seg_page0, seg_page1;        // the page asked for next and the segment's, counted over the block's pages
    int at, e, kvh, first, next_page;      // where the next segment begins; the segment's first page of its sequence
    const int32_t* table;
  } in;
  in.page = warp / CPP;
  in.seg_page0 = in.seg_page1 = 0;
  in.at = u0;
  in.e = e_first;
  in.next_page = -1;
  bool more = true;                        // there are chunks to ask for
  auto look_up = [&]() {                   // the page of the chunk that is asked for next
    while (in.page >= in.seg_page1) {
      if (in.at >= u1) {
        more = false;
        return;
      }
      const Segment s = segment_at(in.at, in.e);
      in.at = s.end;
      in.seg_page0 = in.seg_page1;
      in.seg_page1 += s.n;
      in.kvh = s.kvh;
      in.first = s.d.pg_first + s.first;
      in.table = p.kv.seq_pages + (size_t)s.d.seq * p.kv.pages_stride;
    }
    const int i = in.first + in.page - in.seg_page0;
    in.next_page = i < p.kv.table_pages ? in.table[i] : -1;
  };
  // Where a 16-byte piece lies, so that no two lanes of a load meet in a bank.  Keys in the order of the rows of the product's tile
  // (key r is row 2 (r & 3) + (r >> 2 & 1) of its eight), pieces of odd rows of 128 bytes exchanged; values row by row.  Piece i of a
  // lane is piece lane + 32 i of the chunk: its row and place are the lane's (D = 128: the lane's for even and odd i) and a constant.
  int k_at[2], v_at;
  {
    constexpr int UPR = D / 16;
    const int r = lane / UPR, u = lane % UPR;
    v_at = C::CODES + r * D + (D == 128 ? u ^ ((r & 3) << 1) : u ^ (((r >> 1) & 1) << 1)) * 16;
    if (D == 128) {
      k_at[0] = 2 * r * D + u * 16;
      k_at[1] = (2 * r + 1) * D + (u ^ 4) * 16;
    } else {
      k_at[0] = k_at[1] = (((r & 3) << 1) | (r >> 2)) * D + u * 16;
    }
  }
  int issued = 0;                          // the stage filled next
  auto issue = [&]() {
    if (more) {
      uint8_t* st = ring + issued * C::STAGE;
      const bool known = (unsigned)in.next_page < (unsigned)p.kv.n_pages;
      const size_t row0 = ((size_t)(known ? in.next_page : 0) * Hkv + in.kvh) * PAGE8 + sub * KC;
      const uint8_t* kc = p.k_codes + row0 * D + lane * 16;
      const uint8_t* vc = p.v_codes + row0 * D + lane * 16;
#pragma unroll
      for (int i = 0; i < C::CODES / 512; ++i) {
        cp_async16(st + (D == 128 ? k_at[i & 1] + 1024 * (i >> 1) : k_at[0] + 512 * i), kc + 512 * i, 16);
        cp_async16(st + v_at + 512 * i, vc + 512 * i, 16);
      }
      if (known) {
        if (lane < KC / 2) cp_async16(st + 2 * C::CODES + lane * 16, (lane < KC / 4 ? p.k_scales : p.v_scales - KC) + row0 + lane * 4, 16);
      } else {                             // a page that the pool does not have reads as NaN
        for (int i = lane; i < 2 * KC; i += 32) reinterpret_cast<float*>(st + 2 * C::CODES)[i] = __int_as_float(0x7fffffff);
      }
      in.page += STEP;
      look_up();
    }
    cp_async_commit();
    issued = issued + 1 == STAGES ? 0 : issued + 1;
  };
  look_up();
  pdl_wait();
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue();
  int mine[2] = {0, 0};                    // whose partial results the block leaves

  // ---- segments: the block's part of one (entry, kv head) after the other ----
  int taken = 0;                           // the stage read next
  int page = warp / CPP, seg_page0 = 0;    // the page of the chunk in it and the segment's first, counted over the block's pages
  int e = e_first;
  for (int at_unit = u0; at_unit < u1;) {
    const Segment s = segment_at(at_unit, e);
    const Rw8Entry& d = s.d;
    const int kvh = s.kvh;
    at_unit = s.end;
    if (s.n <= 0) continue;                // (the range ends among the units of no page)

    // neg: -M, 0 while there is no M; Lc: what L has too much (32-bit path)
    float O[KS][NT][4], M[NT][2], neg[NT][2], L[NT][2], Lc[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int j = 0; j < 2; ++j) M[n][j] = -INFINITY, neg[n][j] = L[n][j] = Lc[n][j] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) O[i][n][j] = 0.f;
    }
    // queries: row n * 8 + g, its dims in the order in which a lane has the keys' codes
    uint32_t qf[SP][NT][KS][2];
    float fac[NT][2];                      // of the columns 2t, 2t + 1: scale * log2(e) * the row's power of two
    int col_pos[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = n * 8 + g;
      float x[D / 4];
      float a = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const int row = d.row0 + r;
        const size_t at = (size_t)(d.q_start + row / G) * p.ldq + (size_t)(kvh * G + row % G) * D + 64 * c + 16 * t;
        if (SP == 1 && !p.q_f32) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint4 raw = make_uint4(0u, 0u, 0u, 0u);
            if (r < d.rows) raw = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)p.q + at + 8 * h);
            const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = __bfloat1622float2(b[i]);
              x[c * 16 + h * 8 + 2 * i] = f.x;
              x[c * 16 + h * 8 + 2 * i + 1] = f.y;
            }
          }
        } else {
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < d.rows) f = *reinterpret_cast<const float4*>((const float*)p.q + at + 4 * h);
            x[c * 16 + 4 * h] = f.x, x[c * 16 + 4 * h + 1] = f.y, x[c * 16 + 4 * h + 2] = f.z, x[c * 16 + 4 * h + 3] = f.w;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < D / 4; ++i) a = fmaxf(a, fabsf(x[i]));
      a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
      a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
      // times a power of two that brings the row's largest entry between 2^14 and 2^15 (rows that are zero or not finite: 2^15)
      int ex = 0;
      if (a > 0.f && a <= FLT_MAX) ex = max(-100, (int)((__float_as_uint(a) >> 23) & 255) - 126);
      const float down = __uint_as_float((uint32_t)(127 + 15 - ex) << 23);
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float y0 = x[4 * s + 2 * h] * down, y1 = x[4 * s + 2 * h + 1] * down;
          const __half2 hi = __floats2half2_rn(y0, y1);
          qf[0][n][s][h] = as_u32(hi);
          if (SP == 2) qf[SP - 1][n][s][h] = pack_half2(y0 - __low2float(hi), y1 - __high2float(hi));
        }
      const float f = ldexpf(p.scale_log2, ex - 15);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        fac[n][j] = __shfl_sync(0xffffffffu, f, (2 * t + j) * 4);
        const int r2 = n * 8 + 2 * t + j;
        col_pos[n][j] = d.pos0 + (d.row0 + min(r2, d.rows - 1)) / G;
      }
    }
    const int first_pos = d.pos0 + d.row0 / G;
    bool unset = true;                     // some column has no maximum yet

    auto chunk = [&](auto masked_c, const uint8_t* st, int key0) {
      constexpr bool MASKED = decltype(masked_c)::value;
      const float* ks_s = reinterpret_cast<const float*>(st + 2 * C::CODES);
      const float* vs_s = ks_s + KC;
      float S[MT][NT][4], vs[MT][2], ks[MT][2];
      uint32_t hidden = 0u;                // bit (m * NT + n) * 4 + j: that score's key is not seen
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
          for (int j = 0; j < 4; ++j) S[m][n][j] = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          uint32_t a[4];
          halves8x4<HELD>(ka[s], a[0], a[2]);
          halves8x4<HELD>(kb[s], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int z = 0; z < SP; ++z) mma_f16(S[m][n], a, qf[z][n][s][0], qf[z][n][s][1]);
        }
        // rows g and g + 8 of the tile are the keys pk and pk + 8
        const int pk = m * 16 + (g >> 1) + 4 * (g & 1);
        ks[m][0] = ks_s[pk], ks[m][1] = ks_s[pk + 8];
        vs[m][0] = vs_s[pk], vs[m][1] = vs_s[pk + 8];
        if (MASKED) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = key0 + pk + (j < 2 ? 0 : 8);
              if (key > col_pos[n][j & 1] || (p.window > 0 && key <= col_pos[n][j & 1] - p.window)) hidden |= 1u << ((m * NT + n) * 4 + j);
            }
        }
      }
      auto is_hidden = [&](int m, int n, int j) { return MASKED && ((hidden >> ((m * NT + n) * 4 + j)) & 1u); };
      uint32_t pb[SP][MT][NT][2];
      float sum[NT][2];
      auto weigh = [&]() {                 // weights, packed for the second product, and their sums; -> whether they are in range
        __half2 top = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
        bool fine = true;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          sum[n][0] = SP == 2 ? 0.f : L[n][0], sum[n][1] = SP == 2 ? 0.f : L[n][1];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            float w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x = fast_exp2(fmaf(S[m][n][j], ks[m][j >> 1] * fac[n][j & 1], neg[n][j & 1]));
              w[j] = x * vs[m][j >> 1];
              if (is_hidden(m, n, j)) x = 0.f, w[j] = 0.f;               // (the key's scales may be anything)
              sum[n][j & 1] += x;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const __half2 hi = __floats2half2_rn(w[2 * h], w[2 * h + 1]);
              top = __hmax2(top, hi);
              pb[0][m][n][h] = as_u32(hi);
              if (SP == 2) pb[SP - 1][m][n][h] = pack_half2((w[2 * h] - __low2float(hi)) * 2048.f, (w[2 * h + 1] - __high2float(hi)) * 2048.f);
            }
          }
          fine = fine && !((SP == 2 ? L[n][0] : 0.f) + sum[n][0] > RW8_SUM) && !((SP == 2 ? L[n][1] : 0.f) + sum[n][1] > RW8_SUM);
        }
        return fine && !(fmaxf(__low2float(top), __high2float(top)) > RW8_LAZY);
      };
      const bool fine = weigh();
      if (__any_sync(0xffffffffu, unset || !fine)) {
        unset = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = -INFINITY;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (!is_hidden(m, n, j + 2 * h)) mx = fmaxf(mx, S[m][n][j + 2 * h] * (ks[m][h] * fac[n][j]) + fast_log2(fmaxf(vs[m][h], RW8_TINY)));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(M[n][j], mx - RW8_UP), f = M[n][j] == -INFINITY ? 1.f : fast_exp2(M[n][j] - m_new);
            if (M[n][j] != -INFINITY) {
              L[n][j] = rescale8(L[n][j], M[n][j] - m_new);
              if (SP == 2) Lc[n][j] = rescale8(Lc[n][j], M[n][j] - m_new);
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) O[i][n][j] *= f, O[i][n][j + 2] *= f;
            M[n][j] = m_new;
            neg[n][j] = m_new == -INFINITY ? 0.f : -m_new;
            unset = unset || m_new == -INFINITY;
          }
        unset = __any_sync(0xffffffffu, unset);
        weigh();
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (SP == 2) {
            const float x = sum[n][j] - Lc[n][j], l = L[n][j] + x;
            Lc[n][j] = (l - L[n][j]) - x;
            L[n][j] = l;
          } else {
            L[n][j] = sum[n][j];
          }
        }
      const int seen0 = max(d.lo - key0, 0), seen1 = d.last - key0;      // rows of the chunk that some query sees
#pragma unroll
      for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int z = 0; z < SP; ++z)
#pragma unroll
          for (int n = 0; n < NT; ++n) pb[z][m][n][0] = transpose8x8(pb[z][m][n][0]), pb[z][m][n][1] = transpose8x8(pb[z][m][n][1]);
        // values: keys 2t, 2t + 1 (+ 8) of the tile are the rows t, t + 4 (+ 8); a lane has the dims g * D / 8 ..
        uint32_t vw[4][D / 32];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = m * 16 + t + 4 * (j & 1) + 8 * (j >> 1);
          if (D == 128) {
            const uint4 v = *reinterpret_cast<const uint4*>(st + C::CODES + r * D + ((g ^ ((r & 3) << 1)) * 16));
            vw[j][0] = v.x, vw[j][1] = v.y, vw[j][D / 32 - 2] = v.z, vw[j][D / 32 - 1] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(st + C::CODES + r * D + (((g >> 1) ^ (((r >> 1) & 1) << 1)) * 16) + (g & 1) * 8);
            vw[j][0] = v.x, vw[j][1] = v.y;
          }
          if (MASKED && (r < seen0 || r > seen1)) {                      // (what lies there may be no number)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) vw[j][i] = 0u;
          }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {       // four dims: two tiles of dims
          uint32_t z4[4], a01[4], a23[4];
          asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(z4[0]) : "r"(vw[0][w]), "r"(vw[1][w]));
          asm("prmt.b32 %0, %1, %2, 0x7362;" : "=r"(z4[1]) : "r"(vw[0][w]), "r"(vw[1][w]));
          asm("prmt.b32 %0, %1, %2, 0x5140;" : "=r"(z4[2]) : "r"(vw[2][w]), "r"(vw[3][w]));
          asm("prmt.b32 %0, %1, %2, 0x7362;" : "=r"(z4[3]) : "r"(vw[2][w]), "r"(vw[3][w]));
          halves8x4<HELD>(z4[0], a01[0], a01[1]);
          halves8x4<HELD>(z4[2], a01[2], a01[3]);
          halves8x4<HELD>(z4[1], a23[0], a23[1]);
          halves8x4<HELD>(z4[3], a23[2], a23[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (SP == 2) {
              float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(c0, a01, pb[SP - 1][m][n][0], pb[SP - 1][m][n][1]);
              mma_f16(c1, a23, pb[SP - 1][m][n][0], pb[SP - 1][m][n][1]);
#pragma unroll
              for (int j = 0; j < 4; ++j) c0[j] *= 1.f / 2048.f, c1[j] *= 1.f / 2048.f;
              mma_f16(c0, a01, pb[0][m][n][0], pb[0][m][n][1]);
              mma_f16(c1, a23, pb[0][m][n][0], pb[0][m][n][1]);
#pragma unroll
              for (int j = 0; j < 4; ++j) O[2 * w][n][j] += c0[j], O[2 * w + 1][n][j] += c1[j];
            } else {
              mma_f16(O[2 * w][n], a01, pb[0][m][n][0], pb[0][m][n][1]);
              mma_f16(O[2 * w + 1][n], a23, pb[0][m][n][0], pb[0][m][n][1]);
            }
          }
        }
      }
    };

    for (; page < seg_page0 + s.n; page += STEP) {
      cp_async_wait<STAGES - 2>();
      __syncwarp();                        // every lane's copies are here, and every lane is done with the stage before
      issue();
      const uint8_t* st = ring + taken * C::STAGE;
      taken = taken + 1 == STAGES ? 0 : taken + 1;
      const int key0 = (d.pg_first + s.first + page - seg_page0) * PAGE8 + sub * KC;
      if (key0 + KC - 1 > first_pos || (p.window > 0 && key0 <= d.last - p.window)) chunk(std::true_type{}, st, key0);
      else chunk(std::false_type{}, st, key0);
    }
    seg_page0 += s.n;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (SP == 2) L[n][j] -= Lc[n][j];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) L[n][j] += __shfl_xor_sync(0xffffffffu, L[n][j], o);
      }

    // ---- the warps' states meet: each leaves its own where nothing is being copied to (the stage read last; `issue` fills the one
    // before it first), then a warp has some tiles of the output from all eight ----
    auto state_of = [&](int w, int stage) { return reinterpret_cast<float*>(C::IN_RING ? smem + (w * STAGES + stage) * C::STAGE : smem + C::RING + w * C::STATE); };
    __shared__ uint8_t s_stage[RW8_WARPS];
    {
      __syncwarp();
      const int free_stage = taken == 0 ? STAGES - 1 : taken - 1;
      if (lane == 0) s_stage[warp] = (uint8_t)free_stage;
      float* at = state_of(warp, free_stage);
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) at[((i * NT + n) * 4 + j) * 32 + lane] = O[i][n][j];
      if (g == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) at[C::PAIRS * 128 + n * 8 + 2 * t + j] = M[n][j], at[C::PAIRS * 128 + 8 * NT + n * 8 + 2 * t + j] = L[n][j];
      }
    }
    __syncthreads();
    // other blocks have pages of it too: a partial result, of the block's first segment or of its last
    const bool shared_out = s.n < d.n_pages;
    const int part = u0 < s.begin ? 1 : 0;
    float* my_slot = p.slots + (size_t)(2 * blockIdx.x + part) * C::SLOT;
    if (shared_out) {
      const int id = ((s.number * Hkv + kvh + 1) << 1) | (s.first == 0 ? 1 : 0);
      if (part) mine[1] = id;
      else mine[0] = id;
    }
    auto store = [&](float* slot, int pair, const Rw8Tile& r) {
#pragma unroll
      for (int j = 0; j < 4; ++j) __stcg(slot + (pair * 4 + j) * 32 + lane, r.o[j]);
      if (pair < NT && g == 0) {
#pragma unroll
        for (int j = 0; j < 2; ++j) __stcg(slot + C::PAIRS * 128 + pair * 8 + 2 * t + j, r.m[j]), __stcg(slot + C::PAIRS * 128 + 8 * NT + pair * 8 + 2 * t + j, r.l[j]);
      }
    };
    for (int pair = warp; pair < C::PAIRS; pair += RW8_WARPS) {
      const Rw8Tile r = rw8_gather<C, NT>(pair, 0, RW8_WARPS, 1, [&](int w) { return (const float*)state_of(w, s_stage[w]); }, [](const float* x) { return *x; });
      if (shared_out) store(my_slot, pair, r);
      else rw8_write<D, NT, T>(p, d, kvh, pair, r);
    }
    __syncthreads();                       // the stages may be filled again, s_stage written
  }
  cp_async_wait_all();
  if (threadIdx.x < 2) p.whose[2 * blockIdx.x + threadIdx.x] = mine[threadIdx.x];
}

// The (entry, kv head)s that several blocks have pages of: block c joins the one whose first part block c of the kernel above left.
template <int D, int NT, typename T> __global__ void __launch_bounds__(RW8_WARPS * 32) rows8_join_kernel(Rows8Params p) {
  using C = Rw8Cfg<D, NT, T>;
  constexpr int SHARE = C::PAIRS < RW8_WARPS ? RW8_WARPS / C::PAIRS : 1;      // warps that share a tile's parts
  __shared__ float s_tile[RW8_WARPS][256];
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int last = (int)gridDim.x - 1, w0 = p.whose[2 * c], w1 = p.whose[2 * c + 1];
  int next = p.whose[2 * min(c + 1 + lane, last)];         // (asked for with the others: the loads are the kernel's time)
  const int which = (w1 & 1) ? 1 : 0, id = which ? w1 : w0;
  if (!(id & 1)) return;
  int n_parts = 1;
  for (int z0 = c + 1;; z0 += 32) {
    const uint32_t other = __ballot_sync(0xffffffffu, z0 + lane > last || next != id - 1);
    n_parts += other ? __ffs(other) - 1 : 32;
    if (other) break;
    next = p.whose[2 * min(z0 + 32 + lane, last)];
  }
  const int pair_id = (id >> 1) - 1, number = pair_id / p.kv.n_kv_heads, kvh = pair_id - number * p.kv.n_kv_heads;
  const Rw8Entry d = rw8_entry(p, number, 8 * NT);
  for (int pair = warp / SHARE; pair < C::PAIRS; pair += RW8_WARPS / SHARE) {
    Rw8Tile r = rw8_gather<C, NT>(pair, warp % SHARE, n_parts, SHARE,
                                  [&](int z) { return (const float*)(p.slots + (size_t)(2 * (c + z) + (z == 0 ? which : 0)) * C::SLOT); },
                                  [](const float* x) { return *x; });
    if (SHARE > 1) {                       // (once through the loop)
      float* mine = s_tile[warp] + lane;
      mine[0] = r.o[0], mine[32] = r.o[1], mine[64] = r.o[2], mine[96] = r.o[3], mine[128] = r.m[0], mine[160] = r.m[1], mine[192] = r.l[0], mine[224] = r.l[1];
      __syncthreads();
      if (warp % SHARE) return;
#pragma unroll
      for (int w = 1; w < SHARE; ++w) {
        const float* x = s_tile[warp + w] + lane;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float m = x[128 + 32 * j], top = fmaxf(r.m[j], m);
          const float f = r.m[j] == -INFINITY ? 0.f : r.m[j] - top, h = m == -INFINITY ? 0.f : m - top;
          r.l[j] = rescale8(r.l[j], f) + rescale8(x[192 + 32 * j], h);
          r.m[j] = top;
          r.o[j] = r.o[j] * fast_exp2(f) + x[32 * j] * fast_exp2(h);
          r.o[j + 2] = r.o[j + 2] * fast_exp2(f) + x[64 + 32 * j] * fast_exp2(h);
        }
      }
    }
    rw8_write<D, NT, T>(p, d, kvh, pair, r);
  }
}

template <int D, int NT, int HELD, typename T> int launch_rows8(const Rows8Params& p, int n_entries, int grid, int most_pages, cudaStream_t stream) {
  using C = Rw8Cfg<D, NT, T>;
  constexpr auto kernel = attention_rows8_kernel<D, NT, HELD, T>;
  static PerDevice<bool> configured;
  if (!configured.here()) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::RING + C::MERGE + 6 * (RW8_MAX_ENTRIES + 1)) != cudaSuccess)
      return LLMI_ERR_LAUNCH;
    configured.here() = true;
  }
  const size_t smem = C::RING + C::MERGE + 4 * ((size_t)n_entries + 1) + (p.row_tiles > 1 ? 2 * ((size_t)p.n_seqs + 1) : 0);
  // no more blocks than are resident: many entries' table may leave room for one a SM only (228 KB; a block's own 1 KB and its statics)
  const int fit = (int)((228 << 10) / (smem + 1280));
  grid = min(grid, min(C::BLOCKS, max(1, fit)) * sm_count());
  const Rw8Cut cut = {8, 1024 / D + 1, 512 / D, 256 / D};
  const int rc = launch_pdl(PDL_ATTENTION, kernel, (unsigned)grid, RW8_WARPS * 32, smem, stream, p, n_entries, cut);
  // (short (entry, kv head)s that have a block each leave no parts)
  if (rc != LLMI_OK || ((long)n_entries * p.kv.n_kv_heads <= grid && most_pages <= cut.most_whole)) return rc;
  return launch_pdl(PDL_ATTENTION, rows8_join_kernel<D, NT, T>, (unsigned)grid, RW8_WARPS * 32, 0, stream, p);
}

// Eighths of query rows in a tile: the fewest that hold a sequence's rows, of those there are.
inline int rw8_tiles(int dtype, int D, long rows) {
  if (dtype == LLMI_DTYPE_F32) return rows <= 8 || D == 128 ? 1 : 2;
  return rows <= 8 ? 1 : (rows <= 16 || D == 128) ? 2 : 4;
}
// Row tiles that a sequence of `max_q` tokens has; entries that a call has at most: the tiles of all sequences, each of which may leave
// its last one all but empty, or (one tile a sequence) a sequence each.
inline long rw8_row_tiles(int nt, int max_q, int group) { return ((long)max_q * group + 8 * nt - 1) / (8 * nt); }
inline long rw8_entries(int nt, int n_tokens, int n_seqs, long tiles, int group) {
  const long all = n_seqs * tiles, there = ((long)n_tokens * group + (8L * nt - 1) * n_seqs) / (8 * nt);
  return tiles == 1 || all < there ? all : there;
}
inline int rw8_grid(long units) { return (int)(units < 2L * sm_count() ? units : 2L * sm_count()); }

}  // namespace llmi

using namespace llmi;

// The floats of scratch for the blocks' partial results (of any content); below 0: the sizes are not taken.  `n_tokens`: at least those of
// all sequences; `max_q`: most tokens that a sequence brings.
LLMI_EXPORT long llmi_attention_rows8_workspace(int dtype, int n_tokens, int n_seqs, int max_q, int n_heads, int n_kv_heads, int head_dim, int table_pages) {
  if (n_tokens <= 0 || n_seqs <= 0 || max_q <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || (head_dim != 64 && head_dim != 128) || table_pages <= 0)
    return LLMI_ERR_BAD_SIZE;
  const int group = n_heads / n_kv_heads, nt = rw8_tiles(dtype, head_dim, (long)max_q * group);
  const long tiles = rw8_row_tiles(nt, max_q, group), entries = rw8_entries(nt, n_tokens, n_seqs, tiles, group);
  if (entries > RW8_MAX_ENTRIES || n_seqs > RW8_MAX_ENTRIES || n_seqs * tiles * n_kv_heads > 0x3ffffff0L ||
      entries * n_kv_heads * ((long)table_pages + 64) > 0x7fffffffL)
    return LLMI_ERR_BAD_SIZE;
  return 2L * rw8_grid(entries * n_kv_heads * (long)table_pages) * (head_dim / 16 * nt * 128 + 16 * nt + 1);
}

LLMI_EXPORT int llmi_attention_rows8(int dtype, int held, const void* q, long ldq, void* out, long ldo, const void* k_codes, const float* k_scales,
                                     const void* v_codes, const float* v_scales, const int32_t* seq_q_start, const int32_t* seq_kv_len,
                                     const int32_t* seq_pages, int pages_stride, int table_pages, int n_seqs, int n_pages, int n_tokens,
                                     int max_q, int n_heads, int n_kv_heads, int head_dim, float scale, int window, int q_f32, float* slots, long n_floats,
                                     cudaStream_t stream) {
  if (dtype != LLMI_DTYPE_F32 && dtype != LLMI_DTYPE_BF16) return LLMI_ERR_BAD_DTYPE;
  const long floats = llmi_attention_rows8_workspace(dtype, n_tokens, n_seqs, max_q, n_heads, n_kv_heads, head_dim, table_pages);
  if (floats < 0 || n_floats < floats || n_pages <= 0 || window < 0) return LLMI_ERR_BAD_SIZE;
  if (held != HELD_INT8 && held != HELD_E4M3) return LLMI_ERR_BAD_DTYPE;
  const long even = dtype == LLMI_DTYPE_F32 ? 3 : 7;         // rows are whole 16-byte pieces
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales) & 15) || (ldq & (q_f32 ? 3 : even)) || (ldo & even))
    return LLMI_ERR_ALIGN;
  const int group = n_heads / n_kv_heads;
  const int nt = rw8_tiles(dtype, head_dim, (long)max_q * group), tiles = (int)rw8_row_tiles(nt, max_q, group);
  Rows8Params p{q, ldq, out, ldo, (const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales,
                seq_q_start, seq_kv_len, Paged8{seq_pages, pages_stride, table_pages, n_pages, n_kv_heads, head_dim}, n_seqs, group, tiles,
                scale * 1.4426950408889634f, window, q_f32, slots, nullptr};
  const int n_entries = (int)rw8_entries(nt, n_tokens, n_seqs, tiles, group), grid = rw8_grid((long)n_entries * n_kv_heads * table_pages);
  p.whose = reinterpret_cast<int*>(slots + 2L * grid * (head_dim / 16 * nt * 128 + 16 * nt));
  // most pages that a (sequence, kv head)'s rows of a tile see
  const long seen = ((long)window + max_q) / PAGE8 + 2;
  const int most_pages = window > 0 && seen <= table_pages ? (int)seen : table_pages + 1;      // (+ 1: page_index8)
#define LLMI_ROWS8(D_, NT_, T_) \
  (held == HELD_INT8 ? launch_rows8<D_, NT_, HELD_INT8, T_>(p, n_entries, grid, most_pages, stream) : launch_rows8<D_, NT_, HELD_E4M3, T_>(p, n_entries, grid, most_pages, stream))
  if (dtype == LLMI_DTYPE_F32) return head_dim == 128 ? LLMI_ROWS8(128, 1, float) : nt == 1 ? LLMI_ROWS8(64, 1, float) : LLMI_ROWS8(64, 2, float);
  if (head_dim == 64) return nt == 1 ? LLMI_ROWS8(64, 1, __nv_bfloat16) : nt == 2 ? LLMI_ROWS8(64, 2, __nv_bfloat16) : LLMI_ROWS8(64, 4, __nv_bfloat16);
  return nt == 1 ? LLMI_ROWS8(128, 1, __nv_bfloat16) : LLMI_ROWS8(128, 2, __nv_bfloat16);
#undef LLMI_ROWS8
}
