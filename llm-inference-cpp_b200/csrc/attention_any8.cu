// Causal grouped-query attention over the paged cache that holds keys and values in 8 bits (rows8.cuh), any sizes, fp32 arithmetic.
//
// For the token t at position pos and query head h, over the keys j of its sequence with lo <= j <= pos (lo = 0, or pos - window + 1
// under a window) and kv head h / (n_heads / n_kv_heads) (reference: src/model/transformer.cpp:263-282):
//     s_j = scale * k_scale[j] * sum_d q[d] * k_code[j][d],   w = softmax(s),   out[d] = sum_j w_j * v_scale[j] * v_code[j][d]
// One warp owns one (token, query head) and takes 32 keys at a time, a key a lane, with a running maximum and sum.
#include <math.h>

#include "rows8.cuh"

namespace llmi {

constexpr int ANY8_WARPS = 4;
constexpr int ANY8_MAX_HD = 256;

struct Any8Params {
  const void* q;
  long ldq;
  void* out;
  long ldo;
  const uint8_t* k_codes;
  const float* k_scales;
  const uint8_t* v_codes;
  const float* v_scales;
  const int32_t* tok_seq;
  const int32_t* tok_pos;
  Paged8 kv;
  int n_tokens, n_seqs, n_heads;
  float scale;
  int window;
  int q_f32;                  // q is fp32 (where out is bf16)
};

template <typename T, int HELD, int NJ>
__global__ void __launch_bounds__(ANY8_WARPS * 32) attention_any8_kernel(Any8Params p) {
  __shared__ float q_s[ANY8_WARPS][ANY8_MAX_HD];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long item = (long)blockIdx.x * ANY8_WARPS + warp;
  const int t = (int)(item / p.n_heads), h = (int)(item - (long)t * p.n_heads);
  if (t >= p.n_tokens) return;
  const int hd = p.kv.head_dim, seq = p.tok_seq[t], pos = p.tok_pos[t];
  if (seq < 0 || seq >= p.n_seqs || pos < 0) return;          // a row of no sequence
  const int kvh = h / (p.n_heads / p.kv.n_kv_heads);
  const int lo = (p.window > 0 && pos - p.window + 1 > 0) ? pos - p.window + 1 : 0;
  const size_t q_at = (size_t)t * p.ldq + (size_t)h * hd;
  for (int d = lane; d < hd; d += 32) q_s[warp][d] = p.q_f32 ? ((const float*)p.q)[q_at + d] : to_f32(((const T*)p.q)[q_at + d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = 0.f;
  for (int c0 = (lo / 32) * 32; c0 <= pos; c0 += 32) {        // (32 keys from a multiple of 32 on lie in one page)
    const int page = page8_of(p.kv, seq, c0);
    if (page < 0) continue;
    const size_t row0 = ((size_t)page * p.kv.n_kv_heads + kvh) * PAGE8 + c0 % PAGE8;
    const int s = c0 + lane;
    const bool valid = s >= lo && s <= pos;
    float score = -INFINITY, vs = 0.f;
    if (valid) {
      const uint8_t* k = p.k_codes + (row0 + lane) * hd;
      float dot = 0.f;
      for (int d = 0; d < hd; ++d) dot = fmaf(q_s[warp][d], code8<HELD>(k[d]), dot);
      score = dot * p.k_scales[row0 + lane] * p.scale;
      vs = p.v_scales[row0 + lane];
    }
    const float m_new = fmaxf(m, warp_max(score));
    const float base = m_new == -INFINITY ? 0.f : m_new;      // (scores of -infinity only: nothing to weigh yet)
    const float w = valid ? expf(score - base) : 0.f;
    const float corr = expf(m - base);
    l = l * corr + warp_sum(w);
    const float wv = valid ? w * vs : 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] *= corr;
    const int first = max(lo - c0, 0), last = min(pos - c0, 31);
    for (int kk = first; kk <= last; ++kk) {
      const float pk = __shfl_sync(0xffffffffu, wv, kk);
      const uint8_t* v = p.v_codes + (row0 + kk) * hd;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int d = lane + 32 * j;
        if (d < hd) acc[j] = fmaf(pk, code8<HELD>(v[d]), acc[j]);
      }
    }
    m = m_new;
  }
  T* o = (T*)p.out + (size_t)t * p.ldo + (size_t)h * hd;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int d = lane + 32 * j;
    if (d < hd) o[d] = from_f32<T>(l == 0.f ? 0.f : acc[j] / l);      // (0: no page of the sequence is one of the pool)
  }
}

template <typename T, int HELD>
int launch_attention_any8(const Any8Params& p, cudaStream_t stream) {
  const long blocks = ((long)p.n_tokens * p.n_heads + ANY8_WARPS - 1) / ANY8_WARPS;
  if (blocks > 0x7fffffffL) return LLMI_ERR_BAD_SIZE;
  const int nj = (p.kv.head_dim + 31) / 32;
  auto kernel = nj <= 1 ? attention_any8_kernel<T, HELD, 1> : nj <= 2 ? attention_any8_kernel<T, HELD, 2>
              : nj <= 4 ? attention_any8_kernel<T, HELD, 4> : attention_any8_kernel<T, HELD, 8>;
  return launch_pdl(PDL_ATTENTION, kernel, (unsigned)blocks, ANY8_WARPS * 32, 0, stream, p);
}

}  // namespace llmi

using namespace llmi;

LLMI_EXPORT int llmi_attention_any8(int dtype, int held, const void* q, long ldq, void* out, long ldo, const void* k_codes, const float* k_scales,
                                    const void* v_codes, const float* v_scales, const int32_t* tok_seq, const int32_t* tok_pos,
                                    const int32_t* seq_pages, int pages_stride, int table_pages, int n_seqs, int n_pages, int n_tokens,
                                    int n_heads, int n_kv_heads, int head_dim, float scale, int window, int q_f32, cudaStream_t stream) {
  if (n_tokens <= 0 || n_seqs <= 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads || head_dim <= 0 || head_dim > ANY8_MAX_HD ||
      n_pages <= 0 || window < 0)
    return LLMI_ERR_BAD_SIZE;
  if (held != HELD_INT8 && held != HELD_E4M3) return LLMI_ERR_BAD_DTYPE;
  Any8Params p{q, ldq, out, ldo, (const uint8_t*)k_codes, k_scales, (const uint8_t*)v_codes, v_scales, tok_seq, tok_pos,
               Paged8{seq_pages, pages_stride, table_pages, n_pages, n_kv_heads, head_dim}, n_tokens, n_seqs, n_heads, scale, window, q_f32};
  if (dtype == LLMI_DTYPE_F32)
    return held == HELD_INT8 ? launch_attention_any8<float, HELD_INT8>(p, stream) : launch_attention_any8<float, HELD_E4M3>(p, stream);
  if (dtype == LLMI_DTYPE_BF16)
    return held == HELD_INT8 ? launch_attention_any8<__nv_bfloat16, HELD_INT8>(p, stream) : launch_attention_any8<__nv_bfloat16, HELD_E4M3>(p, stream);
  return LLMI_ERR_BAD_DTYPE;
}
