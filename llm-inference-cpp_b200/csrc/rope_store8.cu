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
constexpr int ROPE8_MANY = 256, ROPE8_LANES = 16;      // from so many tokens on, threads of a token beside one another

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
// half of a head and its partner in the second, with the sines and cosines of the pairs between them, and walks over every
// `lanes`-th head of the token; the threads of a head find its maximum by shuffles.  The angle of (position, pair) is the same for
// all heads and sine and cosine are the costly part, so a prompt's threads take several heads (lanes = 16); a decode step's, which is all
// latency, one each.  Bound by bytes: rows read once, q and the codes written once.
template <typename T> struct Piece8;
template <> struct Piece8<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float* f) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  }
  static __device__ __forceinline__ void store(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
template <> struct Piece8<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* f) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = __bfloat1622float2(h[e]);
      f[2 * e] = v.x, f[2 * e + 1] = v.y;
    }
  }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float* f) {
    uint4 raw;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(f[2 * e], f[2 * e + 1]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
};

template <typename T, int HELD>
__global__ void __launch_bounds__(128) rope_store8_rows_kernel(Rope8Params p, int lanes, int log_pieces) {
  constexpr int N = Piece8<T>::N;
  pdl_wait();
  pdl_launch_dependents();
  const int pieces = 1 << log_pieces, per_tok = lanes << log_pieces;       // (pieces divide a warp: a head's threads are neighbours)
  const long item = (long)blockIdx.x * blockDim.x + threadIdx.x;
  const long tok = item / per_tok;
  const int rest = (int)(item - tok * per_tok), hl = rest >> log_pieces, i0 = (rest & (pieces - 1)) * N;
  // (threads without a token go along: the shuffles below are the whole warp's)
  const bool there = tok < p.n_tokens;
  const int t = there ? (int)tok : 0;
  const int seq = p.tok_seq[t], pos = p.tok_pos[t];
  const bool live = there && seq >= 0 && seq < p.n_seqs && pos >= 0;
  const int hd = p.kv.head_dim, half = hd / 2, G = p.kv.n_kv_heads, heads = p.n_heads + (p.write_kv ? 2 * G : 0);
  const int page = live && p.write_kv ? page8_of(p.kv, seq, pos) : -1;
  float sn[N], cs[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    if (p.rotary_dim > 0) sincosf(__fmul_rn((float)pos, p.inv_freq[i0 + e]), &sn[e], &cs[e]);
    else sn[e] = 0.f, cs[e] = 1.f;
  }
  const T* row = (const T*)p.qkv + (size_t)t * p.ld;
#pragma unroll 2
  for (int j0 = 0; j0 < heads; j0 += lanes) {
    const int j = j0 + hl;
    const bool mine = live && j < heads;
    float a[N], b[N], lo[N], hi[N];
    const T* src = row + (size_t)min(j, heads - 1) * hd + i0;
    Piece8<T>::load(src, a);
    Piece8<T>::load(src + half, b);
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
    bool fine = true;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      m = fmaxf(m, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
      fine = fine && finite8(lo[e]) && finite8(hi[e]);
    }
    if (!fine) m = INFINITY;
    for (int o = 1; o < pieces; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    fine = m <= FLT_MAX;
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
    const int lanes = p.n_tokens >= ROPE8_MANY && heads > ROPE8_LANES ? ROPE8_LANES : heads;
    const long n = ((long)p.n_tokens * lanes * pieces + 127) / 128;
    if (n > 0x7fffffffL) return LLMI_ERR_BAD_SIZE;
    return launch_pdl(PDL_ROPE, rope_store8_rows_kernel<T, HELD>, (unsigned)n, 128, 0, stream, p, lanes, log_pieces);
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
