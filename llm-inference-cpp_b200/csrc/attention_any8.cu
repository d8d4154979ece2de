// Causal grouped-query attention over the paged cache that holds keys and values in 8 bits (rows8.cuh), any sizes, fp32 arithmetic.
//
// For the token t at position pos and query head h, over the keys j of its sequence with lo <= j <= pos (lo = 0, or pos - window + 1
// under a window) and kv head h / (n_heads / n_kv_heads) (reference: src/model/transformer.cpp:263-282):
//     s_j = scale * k_scale[j] * sum_d q[d] * k_code[j][d],   w = softmax(s),   out[d] = sum_j w_j * v_scale[j] * v_code[j][d]
// A block owns one (token, query head); warp w takes the keys 32 w .. 32 w + 31 of every 256, a key a lane, with a running maximum and
// sum, and the warps' results are joined in their order: which numbers are added in which order depends on the positions alone, not on
// how a step was cut or batched.  Bound by the latency of a warp's 32 keys (dot products of a lane each, then a row after the other).
// Measured, with 4 codes a load: 16 fp32 tokens over 100 to 1,500 positions, 9 heads by 3 of 64, 56 us (386 with a warp for all keys and
// a code a load); 8 over 4,096, 32 heads by 8 of 96, 272 us; 512 tokens of a prompt, 12 heads by 4 of 96, 155 us.
#include <math.h>

#include "rows8.cuh"

namespace llmi {

constexpr int ANY8_WARPS = 8;
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

// A lane has the dims W (lane + 32 j) .. + W - 1 of a row; W = 4 where rows are whole 4-byte words.
template <typename T, int HELD, int W, int NJ>
__global__ void __launch_bounds__(ANY8_WARPS * 32) attention_any8_kernel(Any8Params p) {
  __shared__ __align__(16) float q_s[ANY8_MAX_HD];
  __shared__ float s_acc[ANY8_WARPS][ANY8_MAX_HD], s_m[ANY8_WARPS], s_l[ANY8_WARPS];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = (int)(blockIdx.x / (unsigned)p.n_heads), h = (int)(blockIdx.x - (unsigned)t * p.n_heads);
  const int hd = p.kv.head_dim, seq = p.tok_seq[t], pos = p.tok_pos[t];
  if (seq < 0 || seq >= p.n_seqs || pos < 0) return;          // a row of no sequence
  const int kvh = h / (p.n_heads / p.kv.n_kv_heads);
  const int lo = (p.window > 0 && pos - p.window + 1 > 0) ? pos - p.window + 1 : 0;
  const size_t q_at = (size_t)t * p.ldq + (size_t)h * hd;
  for (int d = threadIdx.x; d < hd; d += ANY8_WARPS * 32) q_s[d] = p.q_f32 ? ((const float*)p.q)[q_at + d] : to_f32(((const T*)p.q)[q_at + d]);
  __syncthreads();
  auto codes = [](const uint8_t* at, float (&x)[W]) {
    if (W == 4) {
      uint32_t a, b;
      halves8x4<HELD>(*reinterpret_cast<const uint32_t*>(at), a, b);
      const float2 f = __half22float2(*reinterpret_cast<__half2*>(&a)), g = __half22float2(*reinterpret_cast<__half2*>(&b));
      x[0] = f.x, x[W - 3] = f.y, x[W - 2] = g.x, x[W - 1] = g.y;
    } else {
      x[0] = code8<HELD>(*at);
    }
  };
  float m = -INFINITY, l = 0.f, acc[NJ][W];
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < W; ++i) acc[j][i] = 0.f;
  constexpr int ROUND = ANY8_WARPS * 32;
  // (32 keys from a multiple of 32 on lie in one page)
  for (long c0 = (long)(lo / ROUND) * ROUND + warp * 32; c0 <= pos; c0 += ROUND) {
    if (c0 + 31 < lo) continue;
    const int page = page8_of(p.kv, seq, (int)c0);
    if (page < 0) {
      l = __int_as_float(0x7fffffff);
      if (c0 / PAGE8 >= p.kv.table_pages) break;
      continue;
    }
    const size_t row0 = ((size_t)page * p.kv.n_kv_heads + kvh) * PAGE8 + c0 % PAGE8;
    const bool valid = c0 + lane >= lo && c0 + lane <= pos;
    float score = -INFINITY, vs = 0.f;
    if (valid) {
      const uint8_t* k = p.k_codes + (row0 + lane) * hd;
      float dot = 0.f;
#pragma unroll 4
      for (int d = 0; d < hd; d += W) {
        float x[W];
        codes(k + d, x);
#pragma unroll
        for (int i = 0; i < W; ++i) dot = fmaf(q_s[d + i], x[i], dot);
      }
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
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < W; ++i) acc[j][i] *= corr;
    const int first = (int)max(lo - c0, 0L), last = (int)min(pos - c0, 31L);
#pragma unroll 4
    for (int kk = first; kk <= last; ++kk) {
      const float pk = __shfl_sync(0xffffffffu, wv, kk);
      const uint8_t* v = p.v_codes + (row0 + kk) * hd;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int d = W * (lane + 32 * j);
        if (d < hd) {
          float x[W];
          codes(v + d, x);
#pragma unroll
          for (int i = 0; i < W; ++i) acc[j][i] = fmaf(pk, x[i], acc[j][i]);
        }
      }
    }
    m = m_new;
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (W * (lane + 32 * j) < hd) s_acc[warp][W * (lane + 32 * j) + i] = acc[j][i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int w = 0; w < ANY8_WARPS; ++w) top = fmaxf(top, s_m[w]);
  if (top == -INFINITY) top = 0.f;
#pragma unroll
  for (int w = 0; w < ANY8_WARPS; ++w) sum += s_l[w] * expf(s_m[w] - top);
  T* o = (T*)p.out + (size_t)t * p.ldo + (size_t)h * hd;
  for (int d = threadIdx.x; d < hd; d += ANY8_WARPS * 32) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < ANY8_WARPS; ++w) x = fmaf(s_acc[w][d], expf(s_m[w] - top), x);
    o[d] = from_f32<T>(x / sum);                  // (scores that are all -infinity: NaN)
  }
}

template <typename T, int HELD>
int launch_attention_any8(const Any8Params& p, cudaStream_t stream) {
  const long blocks = (long)p.n_tokens * p.n_heads;
  if (blocks > 0x7fffffffL) return LLMI_ERR_BAD_SIZE;
  const int hd = p.kv.head_dim;
  const bool words = hd % 4 == 0 && !(((uintptr_t)p.k_codes | (uintptr_t)p.v_codes) & 3);
  auto kernel = words ? (hd <= 128 ? attention_any8_kernel<T, HELD, 4, 1> : attention_any8_kernel<T, HELD, 4, 2>)
              : hd <= 32 ? attention_any8_kernel<T, HELD, 1, 1> : hd <= 64 ? attention_any8_kernel<T, HELD, 1, 2>
              : hd <= 128 ? attention_any8_kernel<T, HELD, 1, 4> : attention_any8_kernel<T, HELD, 1, 8>;
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
