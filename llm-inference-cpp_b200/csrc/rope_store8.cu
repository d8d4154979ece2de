// Rotary position encoding of q and k with the append of k and v to the paged cache that holds them in 8 bits (rows8.cuh says how
// a row is held).  The rotation is rope_store.cu's (rotate-half pairs, angle = float(pos) * inv_freq[i] in fp32; reference formulas:
// src/model/kernels.cpp:122-134, src/model/transformer.cpp:251-262); a rotated key is rounded once, to its codes.
//
// qkv is one row per token: [q heads | k heads | v heads], each head head_dim wide.  Rotated q goes to rows of its own (which may be
// the q part of qkv itself), of qkv's type or fp32 (attention8 asks for those, so that a query is not rounded to bf16 on its way: that
// alone doubles the error of its output); rows of no sequence (tok_seq -1) are left as they are, in q and in the cache.
#include "rows8.cuh"

namespace llmi {

constexpr int ROPE8_MAX_HD = 256;
constexpr int ROPE8_WARPS = 4;
constexpr int ROPE8_THREADS = 512;                     // the most of a block
// Heads of a token that are worked on at a time, each by threads of its own, where all heads would need more threads than the device
// holds (all heads / 16 at a time: 256 tokens of 96 heads of 64 3.5 / 4.3 us, 1,000 of 48 of 128 10.0 / 5.9, 8,192 of 96 62.9 / 34.2).
constexpr int ROPE8_LANES = 16;
constexpr long ROPE8_HELD = 1024;                      // threads a SM

struct Rope8Params {
  const void* qkv;
  long ld;
  void* q_out;
  long ldq;
  const float* inv_freq;
  int rotary_dim;
  const int32_t* tok_seq;
  const int32_t* tok_pos;
  Paged8 kv;
  uint8_t* k_codes;
  float* k_scales;
  uint8_t* v_codes;
  float* v_scales;
  int n_tokens, n_seqs, n_heads, write_kv;
  int q_f32;                  // q_out is fp32 (where qkv is bf16)
};

// Any head size: one warp per (token, head of q, k or v).  The row lies in shared memory as fp32 between its rotation, its maximum
// and its codes.
template <typename T, int HELD>
__global__ void __launch_bounds__(ROPE8_WARPS * 32) rope_store8_kernel(Rope8Params p) {
  __shared__ float rows[ROPE8_WARPS][ROPE8_MAX_HD];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hd = p.kv.head_dim, half = p.rotary_dim / 2;
  const int per_tok = p.n_heads + (p.write_kv ? 2 * p.kv.n_kv_heads : 0);
  const long item = (long)blockIdx.x * ROPE8_WARPS + warp;
  const int t = (int)(item / per_tok), j = (int)(item - (long)t * per_tok);
  if (t >= p.n_tokens) return;
  const int seq = p.tok_seq[t], pos = p.tok_pos[t];
  if (seq < 0 || seq >= p.n_seqs || pos < 0) return;
  const T* src = (const T*)p.qkv + (size_t)t * p.ld + (size_t)j * hd;
  float* row = rows[warp];
  const bool turned = j < p.n_heads + p.kv.n_kv_heads;
  for (int i = lane; i < hd; i += 32) row[i] = to_f32(src[i]);
  __syncwarp();
  if (turned) {
    for (int i = lane; i < half; i += 32) {
      float s, c;
      sincosf(__fmul_rn((float)pos, p.inv_freq[i]), &s, &c);
      const float a = row[i], b = row[i + half];
      row[i] = rot_lo(a, b, c, s);
      row[i + half] = rot_hi(a, b, c, s);
    }
    __syncwarp();
  }
  if (j < p.n_heads) {
    const size_t at = (size_t)t * p.ldq + (size_t)j * hd;
    for (int i = lane; i < hd; i += 32) {
      if (p.q_f32) ((float*)p.q_out)[at + i] = row[i];
      else ((T*)p.q_out)[at + i] = from_f32<T>(row[i]);
    }
    return;
  }
  const int kvh = turned ? j - p.n_heads : j - p.n_heads - p.kv.n_kv_heads;
  const int page = page8_of(p.kv, seq, pos);
  if (page < 0) return;
  float a = 0.f;
  bool finite = true;
  for (int i = lane; i < hd; i += 32) {
    a = fmaxf(a, fabsf(row[i]));
    finite = finite && finite8(row[i]);
  }
  a = warp_max(a);
  finite = __all_sync(0xffffffffu, finite);
  const Scale8 s = scale8<HELD>(a, finite);
  const size_t at = ((size_t)page * p.kv.n_kv_heads + kvh) * PAGE8 + pos % PAGE8;
  uint8_t* codes = (turned ? p.k_codes : p.v_codes) + at * hd;
  for (int i = lane; i < hd; i += 32) codes[i] = (uint8_t)codes8<HELD>(row[i], 0.f, s.inv, finite);
  if (lane == 0) (turned ? p.k_scales : p.v_scales)[at] = s.scale;
}

// Whole-head rotation, or none, of heads that are 2^n 16-byte pieces twice (64, 128 and the like): a thread has one piece of the first
// half of a head and its partner in the second and walks over every `lanes`-th head of the token; the threads of a head find its
// maximum by shuffles.  The angle of (position, pair) is the same for all heads, and sine and cosine are the costly part: a block makes
// each once, in shared memory.  Bound by bytes: rows read once, q and the codes written once.  8,192 tokens of 32 + 64 heads of 64 in
// bf16 take 34 us, 5.0 TB/s (with the sines in every thread 43); 3,500 of 15 + 10 in fp32 14, 3.7 TB/s; a step's few tokens 2.6 to 3.0, a
// kernel's latency.
template <typename T> struct Piece8;
template <> struct Piece8<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void numbers(const uint4& raw, float* f) {
    f[0] = __uint_as_float(raw.x), f[1] = __uint_as_float(raw.y), f[2] = __uint_as_float(raw.z), f[3] = __uint_as_float(raw.w);
  }
  static __device__ __forceinline__ void store(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct Piece8<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void numbers(const uint4& raw, float* f) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) f[2 * e] = __uint_as_float(w[e] << 16), f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* f) {
    uint4 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
};

// The larger in magnitude; NaN where one is.
__device__ __forceinline__ float larger8(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}

template <typename T, int HELD>
__global__ void __launch_bounds__(ROPE8_THREADS) rope_store8_rows_kernel(Rope8Params p, int lanes, int log_pieces, int block_tokens) {
  constexpr int N = Piece8<T>::N;
  extern __shared__ float2 turns[];        // [token][pair]: sine, cosine
  pdl_wait();
  pdl_launch_dependents();
  const int pieces = 1 << log_pieces, per_tok = lanes << log_pieces;       // (pieces divide a warp: a head's threads are neighbours)
  const int own = block_tokens == 1 ? 0 : (int)threadIdx.x / per_tok, rest = (int)threadIdx.x - own * per_tok, hl = rest >> log_pieces;
  const int i0 = (rest & (pieces - 1)) * N;
  const long tok0 = (long)blockIdx.x * block_tokens;
  // (threads without a token go along: the shuffles below are the whole warp's)
  const bool there = own < block_tokens && hl < lanes && tok0 + own < p.n_tokens;
  const int t = (int)(there ? tok0 + own : tok0);
  const int hd = p.kv.head_dim, half = hd / 2, G = p.kv.n_kv_heads, heads = p.n_heads + (p.write_kv ? 2 * G : 0);
  const T* row = (const T*)p.qkv + (size_t)t * p.ld;
  // the rows of a head are under way while the one before is worked on
  uint4 a4 = make_uint4(0u, 0u, 0u, 0u), b4 = a4;
  auto ask = [&](int j) {
    if (!there || j >= heads) return;
    const T* src = row + (size_t)j * hd + i0;
    a4 = *reinterpret_cast<const uint4*>(src), b4 = *reinterpret_cast<const uint4*>(src + half);
  };
  ask(hl);
  const int seq = p.tok_seq[t], pos = p.tok_pos[t];
  const bool live = there && seq >= 0 && seq < p.n_seqs && pos >= 0;
  const int page = live && p.write_kv ? page8_of(p.kv, seq, pos) : -1;
  float sn[N], cs[N];
#pragma unroll
  for (int e = 0; e < N; ++e) sn[e] = 0.f, cs[e] = 1.f;
  if (p.rotary_dim > 0) {
    const int n = (int)min((long)block_tokens, (long)p.n_tokens - tok0) * half;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const int tok = block_tokens == 1 ? 0 : i / half;
      sincosf(__fmul_rn((float)p.tok_pos[tok0 + tok], p.inv_freq[i - tok * half]), &turns[i].x, &turns[i].y);
    }
    __syncthreads();
    if (there) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float2 x = turns[own * half + i0 + e];
        sn[e] = x.x, cs[e] = x.y;
      }
    }
  }
  for (int j0 = 0; j0 < heads; j0 += lanes) {
    const int j = j0 + hl;
    const bool mine = live && j < heads;
    float a[N], b[N], lo[N], hi[N];
    Piece8<T>::numbers(a4, a);
    Piece8<T>::numbers(b4, b);
    ask(j + lanes);
    const bool turned = j < p.n_heads + G && p.rotary_dim > 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      lo[e] = turned ? rot_lo(a[e], b[e], cs[e], sn[e]) : a[e];
      hi[e] = turned ? rot_hi(a[e], b[e], cs[e], sn[e]) : b[e];
    }
    if (mine && j < p.n_heads) {
      const size_t at = (size_t)t * p.ldq + (size_t)j * hd + i0;
      if (sizeof(T) == 2 && p.q_f32) {
        float* dst = (float*)p.q_out + at;
#pragma unroll
        for (int e = 0; e < N; e += 4) Piece8<float>::store(dst + e, lo + e), Piece8<float>::store(dst + half + e, hi + e);
      } else {
        T* dst = (T*)p.q_out + at;
        Piece8<T>::store(dst, lo);
        Piece8<T>::store(dst + half, hi);
      }
    }
    if (j0 + lanes <= p.n_heads) continue;                                 // queries only, for every thread
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) m = larger8(larger8(m, lo[e]), hi[e]);
    for (int o = 1; o < pieces; o <<= 1) m = larger8(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool fine = m <= FLT_MAX;
    if (!mine || j < p.n_heads || page < 0) continue;
    const bool key = j < p.n_heads + G;
    const Scale8 s = scale8<HELD>(m, fine);
    const size_t at = ((size_t)page * G + (key ? j - p.n_heads : j - p.n_heads - G)) * PAGE8 + pos % PAGE8;
    uint8_t* codes = (key ? p.k_codes : p.v_codes) + at * hd + i0;
    uint32_t w[2][N / 4];
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      w[0][e / 4] = codes8<HELD>(lo[e], lo[e + 1], s.inv, fine) | (codes8<HELD>(lo[e + 2], lo[e + 3], s.inv, fine) << 16);
      w[1][e / 4] = codes8<HELD>(hi[e], hi[e + 1], s.inv, fine) | (codes8<HELD>(hi[e + 2], hi[e + 3], s.inv, fine) << 16);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (N == 8) *reinterpret_cast<uint2*>(codes + h * half) = make_uint2(w[h][0], w[h][N / 4 - 1]);
      else *reinterpret_cast<uint32_t*>(codes + h * half) = w[h][0];
    }
    if (i0 == 0) (key ? p.k_scales : p.v_scales)[at] = s.scale;
  }
}

template <typename T, int HELD>
int launch_rope_store8(const Rope8Params& p, cudaStream_t stream) {
  const int pieces = p.kv.head_dim / 2 / Piece8<T>::N, heads = p.n_heads + (p.write_kv ? 2 * p.kv.n_kv_heads : 0);
  if ((p.rotary_dim == p.kv.head_dim || p.rotary_dim == 0) && p.kv.head_dim % (2 * Piece8<T>::N) == 0 && pieces <= 32 && (pieces & (pieces - 1)) == 0 &&
      !(((uintptr_t)p.qkv | (uintptr_t)p.q_out | (uintptr_t)p.k_codes | (uintptr_t)p.v_codes) & 15) && !((p.ld * sizeof(T) | p.ldq * (p.q_f32 ? 4 : sizeof(T))) & 15)) {
    int log_pieces = 0;
    while ((1 << log_pieces) < pieces) ++log_pieces;
    const bool many = (long)p.n_tokens * heads * pieces > ROPE8_HELD * sm_count();
    const int most = many ? ROPE8_LANES : ROPE8_THREADS / pieces, lanes = heads < most ? heads : most;
    const int per_tok = lanes * pieces, block_tokens = per_tok >= 128 ? 1 : 128 / per_tok;
    const int threads = (block_tokens * per_tok + 31) / 32 * 32;
    return launch_pdl(PDL_ROPE, rope_store8_rows_kernel<T, HELD>, (unsigned)((p.n_tokens + block_tokens - 1) / block_tokens), threads,
                      block_tokens * (p.kv.head_dim / 2) * sizeof(float2), stream, p, lanes, log_pieces, block_tokens);
  }
  const long items = (long)p.n_tokens * (p.n_heads + (p.write_kv ? 2 * p.kv.n_kv_heads : 0));
  const long blocks = (items + ROPE8_WARPS - 1) / ROPE8_WARPS;
  if (blocks > 0x7fffffffL) return LLMI_ERR_BAD_SIZE;
  return launch_pdl(PDL_ROPE, rope_store8_kernel<T, HELD>, (unsigned)blocks, ROPE8_WARPS * 32, 0, stream, p);
}

}  // namespace llmi

using namespace llmi;

LLMI_EXPORT int llmi_rope_store8(int dtype, int held, const void* qkv, long ld, void* q_out, long ldq, const float* inv_freq, int rotary_dim,
                                 const int32_t* tok_seq, const int32_t* tok_pos, const int32_t* seq_pages, int pages_stride, int table_pages,
                                 int n_seqs, void* k_codes, float* k_scales, void* v_codes, float* v_scales, int n_pages, int n_tokens,
                                 int n_heads, int n_kv_heads, int head_dim, int write_kv, int q_f32, cudaStream_t stream) {
  if (n_tokens <= 0 || n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || head_dim > ROPE8_MAX_HD || n_pages <= 0)
    return LLMI_ERR_BAD_SIZE;
  if (rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1)) return LLMI_ERR_BAD_SIZE;
  if (held != HELD_INT8 && held != HELD_E4M3) return LLMI_ERR_BAD_DTYPE;
  Rope8Params p{qkv, ld, q_out, ldq, inv_freq, rotary_dim, tok_seq, tok_pos,
                Paged8{seq_pages, pages_stride, table_pages, n_pages, n_kv_heads, head_dim},
                (uint8_t*)k_codes, k_scales, (uint8_t*)v_codes, v_scales, n_tokens, n_seqs, n_heads, write_kv, q_f32};
  if (dtype == LLMI_DTYPE_F32)
    return held == HELD_INT8 ? launch_rope_store8<float, HELD_INT8>(p, stream) : launch_rope_store8<float, HELD_E4M3>(p, stream);
  if (dtype == LLMI_DTYPE_BF16)
    return held == HELD_INT8 ? launch_rope_store8<__nv_bfloat16, HELD_INT8>(p, stream) : launch_rope_store8<__nv_bfloat16, HELD_E4M3>(p, stream);
  return LLMI_ERR_BAD_DTYPE;
}
