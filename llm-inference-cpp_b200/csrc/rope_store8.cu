// Rotary position encoding of q and k with the append of k and v to the paged cache that holds them in 8 bits (rows8.cuh says how
// a row is held).  The rotation is rope_store.cu's (rotate-half pairs, angle = float(pos) * inv_freq[i] in fp32; reference formulas:
// src/model/kernels.cpp:122-134, src/model/transformer.cpp:251-262); a rotated key is rounded once, to its codes.
//
// qkv is one row per token: [q heads | k heads | v heads], each head head_dim wide.  Rotated q goes to rows of its own (which may be
// the q part of qkv itself); rows of no sequence (tok_seq -1) are left as they are, in q and in the cache.
#include "rows8.cuh"

namespace llmi {

constexpr int ROPE8_MAX_HD = 256;
constexpr int ROPE8_WARPS = 4;

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
    T* dst = (T*)p.q_out + (size_t)t * p.ldq + (size_t)j * hd;
    for (int i = lane; i < hd; i += 32) dst[i] = from_f32<T>(row[i]);
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

template <typename T, int HELD>
int launch_rope_store8(const Rope8Params& p, cudaStream_t stream) {
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
                                 int n_heads, int n_kv_heads, int head_dim, int write_kv, cudaStream_t stream) {
  if (n_tokens <= 0 || n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || head_dim > ROPE8_MAX_HD || n_pages <= 0)
    return LLMI_ERR_BAD_SIZE;
  if (rotary_dim < 0 || rotary_dim > head_dim || (rotary_dim & 1)) return LLMI_ERR_BAD_SIZE;
  if (held != HELD_INT8 && held != HELD_E4M3) return LLMI_ERR_BAD_DTYPE;
  Rope8Params p{qkv, ld, q_out, ldq, inv_freq, rotary_dim, tok_seq, tok_pos,
                Paged8{seq_pages, pages_stride, table_pages, n_pages, n_kv_heads, head_dim},
                (uint8_t*)k_codes, k_scales, (uint8_t*)v_codes, v_scales, n_tokens, n_seqs, n_heads, write_kv};
  if (dtype == LLMI_DTYPE_F32)
    return held == HELD_INT8 ? launch_rope_store8<float, HELD_INT8>(p, stream) : launch_rope_store8<float, HELD_E4M3>(p, stream);
  if (dtype == LLMI_DTYPE_BF16)
    return held == HELD_INT8 ? launch_rope_store8<__nv_bfloat16, HELD_INT8>(p, stream) : launch_rope_store8<__nv_bfloat16, HELD_E4M3>(p, stream);
  return LLMI_ERR_BAD_DTYPE;
}
