// Attention of new tokens over the 4-bit key/value cache (format: kv4.cuh):
//   out[t, h, :] = sum_j softmax_j(scale q[t, h, :] . k_j) v_j
// over the keys j <= position of t (causal), or all kv_lens[s] keys of t's
// sequence s, where token t of the last n = cu[s+1] - cu[s] has position
// kv_lens[s] - n + (t - cu[s]).  Query head h reads KV head h / (heads /
// kv_heads).  One pass with the running maximum and sum of the softmax in
// fp32; a row that sees no key is zero.
//
// A block of 128 threads per (token, query head), one page at a time.
#include <cfloat>

#include "kv4.cuh"

namespace cti {
namespace {

using namespace kv4;

struct Args {
  const int32_t* cu;
  const int32_t* kv_lens;
  const int32_t* table;
  int64_t table_stride;
  int table_cols;
  int num_seqs;
  int tokens;
  int heads, kv_heads;
  float scale;
  int causal;
  int64_t num_pages;
  int64_t q_stride;
  int32_t* status;
};

template <typename T, int G>
__global__ void __launch_bounds__(128)
    kv4_attention_kernel(const T* __restrict__ q, const uint8_t* __restrict__ pages, Args a,
                         T* __restrict__ out) {
  using Y = Type16<T>;
  constexpr int D = 32 * G;
  __shared__ float sq[D], part[128], p[64];
  const int t = blockIdx.x, h = blockIdx.y, i = threadIdx.x;
  if (t < __ldg(a.cu) || t >= __ldg(a.cu + a.num_seqs)) return;
  const int s = sequence_of(a.cu, a.num_seqs, t);
  const int64_t len = __ldg(a.kv_lens + s);
  int64_t keys = a.causal ? len - __ldg(a.cu + s + 1) + t + 1 : len;
  if (keys > len) keys = len;
  if (keys > (int64_t)a.table_cols * kPage) {
    if (i == 0) raise_status(a.status, CTI_ERR_BOUNDS, s);
    keys = (int64_t)a.table_cols * kPage;
  }
  const int kvh = h / (a.heads / a.kv_heads);
  if (i < D) {
    const uint16_t bits = reinterpret_cast<const uint16_t*>(q)[t * a.q_stride + h * D + i];
    sq[i] = Y::to_float(bits) * a.scale * 1.4426950408889634f;
  }
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (int64_t j0 = 0; j0 < keys; j0 += kPage) {
    const int64_t page = __ldg(a.table + s * a.table_stride + j0 / kPage);
    if (page < 0 || page >= a.num_pages) {
      if (i == 0) raise_status(a.status, CTI_ERR_BOUNDS, s);
      continue;
    }
    const uint8_t* block = pages + (page * a.kv_heads + kvh) * (int64_t)block_bytes(G);
    __syncthreads();
    const int tau = i & 63, half = i >> 6;
    float dot = 0.0f;
    for (int w = half * 2 * G; w < (half + 1) * 2 * G; ++w) {
      const int g = w >> 2, tt = w & 3;
      uint32_t code = *reinterpret_cast<const uint32_t*>(block + k_word_at(tau, g, tt, G));
      code = __funnelshift_r(code, code, 3);
      const uint32_t meta = *reinterpret_cast<const uint32_t*>(block + k_meta_at(G) +
                                                               k_meta_word_at(tau, g, G));
      for (int e = 0; e < 8; ++e) {
        const int n = (code >> (4 * (e >> 1) + 16 * (e & 1))) & 15;
        dot = fmaf(sq[w * 8 + e], fmaf(16.0f + n, Y::low(meta), Y::high(meta)), dot);
      }
    }
    part[i] = dot;
    __syncthreads();
    const bool seen = j0 + tau < keys;
    const float sc = seen ? part[tau] + part[tau + 64] : -INFINITY;
    __syncthreads();
    if (half == 0) p[tau] = sc;
    __syncthreads();
    float mx = m;
    for (int j = 0; j < 64; ++j) mx = fmaxf(mx, p[j]);
    __syncthreads();
    if (half == 0) p[tau] = seen ? exp2f(sc - mx) : 0.0f;
    __syncthreads();
    const float corr = m == mx ? 1.0f : exp2f(m - mx);
    m = mx;
    l *= corr;
    o *= corr;
    const int last = (int)(keys - j0 < 64 ? keys - j0 : 64);
    for (int j = 0; j < last; ++j) {
      l += p[j];
      if (i < D) {
        const int g = i >> 5, c = (i & 31) >> 2;
        const uint32_t hv = *reinterpret_cast<const uint16_t*>(block + v_codes_at(G) +
                                                               v_half_at(j, g, c, G));
        const uint8_t* vm = block + v_meta_at(G) + v_meta_half_at(j, g, G);
        const float vs = Y::to_float(*reinterpret_cast<const uint16_t*>(vm));
        const float vb = Y::to_float(*reinterpret_cast<const uint16_t*>(vm + 4));
        o = fmaf(p[j], fmaf(16.0f + (float)((hv >> (4 * (i & 3))) & 15), vs, vb), o);
      }
    }
  }
  if (i < D)
    reinterpret_cast<uint16_t*>(out)[((int64_t)t * a.heads + h) * D + i] =
        (uint16_t)Y::bits(l == 0.0f ? 0.0f : o / l);
}

template <typename T, int G>
int launch(const void* q, const void* pages, const Args& a, void* out, cudaStream_t s) {
  kv4_attention_kernel<T, G><<<dim3(a.tokens, a.heads), 128, 0, s>>>(
      static_cast<const T*>(q), static_cast<const uint8_t*>(pages), a, static_cast<T*>(out));
  return cudaGetLastError() == cudaSuccess ? CTI_OK : CTI_ERR_CUDA;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace cti

extern "C" size_t cti_kv4_attention_workspace_bytes(int num_seqs, int64_t tokens, int max_new,
                                                    int64_t max_kv_len, int heads, int kv_heads,
                                                    int head_dim) {
  return 0;
}

extern "C" int cti_kv4_attention(const void* q, int64_t q_stride, int dtype,
                                 const int32_t* cu_seqlens, const int32_t* kv_lens,
                                 const int32_t* page_table, int64_t table_stride, int table_cols,
                                 int num_seqs, int64_t tokens, int max_new, int64_t max_kv_len,
                                 int heads, int kv_heads, int head_dim, float scale, int causal,
                                 const void* pages, int64_t num_pages, void* out, void* workspace,
                                 size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace cti;
  if (num_seqs < 0 || tokens < 0 || max_new < 0 || max_kv_len < 0 || heads <= 0 ||
      kv_heads <= 0 || heads % kv_heads != 0 || num_pages < 0 || table_cols < 0 ||
      !(fabsf(scale) <= FLT_MAX))
    return CTI_ERR_INVALID_ARG;
  if (dtype != CTI_DTYPE_BF16 && dtype != CTI_DTYPE_F16) return CTI_ERR_UNSUPPORTED;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return CTI_ERR_UNSUPPORTED;
  if (tokens > INT32_MAX - 256 || heads > 65535) return CTI_ERR_UNSUPPORTED;
  if (num_seqs == 0 || tokens == 0) return CTI_OK;
  if (!q || !out || !pages || !cu_seqlens || !kv_lens || (!page_table && table_cols > 0))
    return CTI_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(out) || !aligned16(pages)) return CTI_ERR_INVALID_ARG;
  if (q_stride % 8 != 0 || q_stride < (int64_t)heads * head_dim || table_stride < table_cols)
    return CTI_ERR_INVALID_ARG;
  const Args a = {cu_seqlens, kv_lens,  page_table, table_stride, table_cols, num_seqs, (int)tokens,
                  heads,      kv_heads, scale,      causal,       num_pages,  q_stride, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == CTI_DTYPE_BF16)
    return head_dim == 32   ? launch<__nv_bfloat16, 1>(q, pages, a, out, s)
           : head_dim == 64 ? launch<__nv_bfloat16, 2>(q, pages, a, out, s)
                            : launch<__nv_bfloat16, 4>(q, pages, a, out, s);
  return head_dim == 32   ? launch<__half, 1>(q, pages, a, out, s)
         : head_dim == 64 ? launch<__half, 2>(q, pages, a, out, s)
                          : launch<__half, 4>(q, pages, a, out, s);
}
