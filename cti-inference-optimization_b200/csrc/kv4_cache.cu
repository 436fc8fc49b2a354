// Writing tokens into the 4-bit key/value cache and reading them back
// (format: kv4.cuh).
//
// A block takes 32 packed tokens: its first warp finds their pages and
// slots, then every thread takes 8 dims of a token's key and value at a
// time: one 16-byte load each, the four threads of a group share minimum and
// maximum, and each packs its 8 codes.  HBM-bound: 4 + 1.25 bytes per
// element pair (a key's and a value's) either way.
#include <cfloat>

#include "kv4.cuh"

namespace cti {
namespace {

using namespace kv4;

constexpr int kTokens = 32;    // packed tokens of a block
constexpr int kThreads = 256;

struct Args {
  const int32_t* cu;
  const int32_t* kv_lens;
  const int32_t* table;
  int64_t table_stride;
  int table_cols;
  int num_seqs;
  int tokens;
  int kv_heads;
  int64_t num_pages;
  int64_t k_stride, v_stride;
  int32_t* status;
};

CTI_DEVICE float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
CTI_DEVICE float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// The code of x in the group with base b and scale s (inv = 1 / s), exactly:
// k = rint(x / s - b / s) from the reciprocal is at most one off, and only
// where x is within rounding of the border between two codes.  The remainder
// r = (x - b) - (16 + k) s is exact (it is a small difference of numbers on
// the scale's grid), so |r| < s / 2 proves k; else the border decides, with
// the rounding error of x - b taken into account.
CTI_DEVICE int code_of(float x, float b, float s, float inv) {
  const float a = x - b;
  float k = rintf(fmaf(a, inv, -16.0f));
  const float h = 0.5f * s;
  const float r = fmaf(-s, 16.0f + k, a);
  if (fabsf(r) >= h) {
    const float z = a - x;
    const float err = (x - (a - z)) + (-b - z);  // x - b = a + err
    const bool odd = ((int)k & 1) != 0;
    if (r > 0.0f) {
      const float over = (r - h) + err;
      if (over > 0.0f || (over == 0.0f && odd)) k += 1.0f;
    } else {
      const float over = (r + h) + err;
      if (over < 0.0f || (over == 0.0f && odd)) k -= 1.0f;
    }
  }
  return min(max((int)k, 0), 15);
}

// Codes of the 8 values that this thread has of a group of 32 (its quad has
// the others), and the group's scale and base as 16 bits each.
template <typename T>
CTI_DEVICE void quantise8(const uint4& raw, uint32_t (&n)[8], uint32_t& s_bits, uint32_t& b_bits) {
  using Y = Type16<T>;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Y::low(w[i]);
    x[2 * i + 1] = Y::high(w[i]);
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  // The scale is rounded to T from fp32; max - min and the quotient are
  // nearer to the true value than any T border that they could cross.
  s_bits = Y::bits((hi - lo) / 15.0f);
  float s = Y::to_float(s_bits);
  if (s < FLT_MIN) {  // below the smallest normal fp32 number: a constant group
    s = 0.0f;
    s_bits = 0;
  }
  b_bits = Y::bits(fmaf(-16.0f, s, lo));
  const float b = Y::to_float(b_bits);
  if (!(fabsf(b) <= FLT_MAX) || !(s <= FLT_MAX)) {
    s_bits = b_bits = 0x7fffu;  // NaN in both types
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = 0;
    return;
  }
  const float inv = s > 0.0f ? 1.0f / s : 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = s > 0.0f ? (uint32_t)code_of(x[i], b, s, inv) : 0u;
}

CTI_DEVICE void find_places(const Args& a, int t0, Place (&places)[kTokens]) {
  if (threadIdx.x < kTokens) {
    const int t = t0 + threadIdx.x;
    Place at = {-1, 0};
    if (t < a.tokens && a.num_seqs > 0 && t >= __ldg(a.cu) && t < __ldg(a.cu + a.num_seqs))
      at = place_of(a.cu, a.kv_lens, a.table, a.table_stride, a.table_cols, a.num_seqs,
                    a.num_pages, t, a.status);
    else
      at.page = -2;  // of no sequence
    places[threadIdx.x] = at;
  }
  __syncthreads();
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads)
    kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, Args a,
                      uint8_t* __restrict__ pages) {
  __shared__ Place places[kTokens];
  const int t0 = blockIdx.x * kTokens;
  find_places(a, t0, places);
  const int per = a.kv_heads * G * 4;  // 8-dim pieces of a token
  const int total = kTokens * per;     // a multiple of 32
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int tok = i / per, piece = i - tok * per;
    const Place at = places[tok];
    const int head = piece / (4 * G), g = (piece >> 2) & (G - 1), t = piece & 3;
    const bool live = at.page >= 0;
    uint4 rk = make_uint4(0, 0, 0, 0), rv = rk;
    if (live) {
      rk = __ldg(reinterpret_cast<const uint4*>(k + (t0 + tok) * a.k_stride + piece * 8));
      rv = __ldg(reinterpret_cast<const uint4*>(v + (t0 + tok) * a.v_stride + piece * 8));
    }
    uint32_t nk[8], nv[8], ks, kb, vs, vb;
    quantise8<T>(rk, nk, ks, kb);
    quantise8<T>(rv, nv, vs, vb);
    if (!live) continue;  // the loop's bound is the same for a whole warp
    uint8_t* block = pages + (at.page * a.kv_heads + head) * (int64_t)block_bytes(G);
    uint32_t wk = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) wk |= nk[2 * j] << (4 * j) | nk[2 * j + 1] << (16 + 4 * j);
    *reinterpret_cast<uint32_t*>(block + k_word_at(at.slot, g, t, G)) = __funnelshift_l(wk, wk, 3);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t hv = nv[4 * c] | nv[4 * c + 1] << 4 | nv[4 * c + 2] << 8 | nv[4 * c + 3] << 12;
      *reinterpret_cast<uint16_t*>(block + v_codes_at(G) + v_half_at(at.slot, g, 2 * t + c, G)) =
          (uint16_t)hv;
    }
    if (t == 0) {
      *reinterpret_cast<uint32_t*>(block + k_meta_at(G) + k_meta_word_at(at.slot, g, G)) =
          ks | kb << 16;
      uint8_t* vm = block + v_meta_at(G) + v_meta_half_at(at.slot, g, G);
      *reinterpret_cast<uint16_t*>(vm) = (uint16_t)vs;
      *reinterpret_cast<uint16_t*>(vm + 4) = (uint16_t)vb;
    }
  }
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads)
    kv4_read_kernel(const uint8_t* __restrict__ pages, Args a, T* __restrict__ k,
                    T* __restrict__ v) {
  using Y = Type16<T>;
  __shared__ Place places[kTokens];
  const int t0 = blockIdx.x * kTokens;
  find_places(a, t0, places);
  const int per = a.kv_heads * G * 4;
  const int total = kTokens * per;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int tok = i / per, piece = i - tok * per;
    const Place at = places[tok];
    if (at.page == -2) continue;
    const int head = piece / (4 * G), g = (piece >> 2) & (G - 1), t = piece & 3;
    uint4 ok = make_uint4(0, 0, 0, 0), ov = ok;
    if (at.page >= 0) {
      const uint8_t* block = pages + (at.page * a.kv_heads + head) * (int64_t)block_bytes(G);
      uint32_t wk = __ldg(reinterpret_cast<const uint32_t*>(block + k_word_at(at.slot, g, t, G)));
      wk = __funnelshift_r(wk, wk, 3);
      const uint32_t mk = __ldg(
          reinterpret_cast<const uint32_t*>(block + k_meta_at(G) + k_meta_word_at(at.slot, g, G)));
      const uint8_t* vm = block + v_meta_at(G) + v_meta_half_at(at.slot, g, G);
      const float ks = Y::low(mk), kb = Y::high(mk);
      const float vs = Y::to_float(__ldg(reinterpret_cast<const uint16_t*>(vm)));
      const float vb = Y::to_float(__ldg(reinterpret_cast<const uint16_t*>(vm + 4)));
      uint32_t o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = Y::pack(fmaf(16.0f + (float)((wk >> (4 * j)) & 15), ks, kb),
                       fmaf(16.0f + (float)((wk >> (16 + 4 * j)) & 15), ks, kb));
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t hv = __ldg(reinterpret_cast<const uint16_t*>(
            block + v_codes_at(G) + v_half_at(at.slot, g, 2 * t + c, G)));
#pragma unroll
        for (int j = 0; j < 2; ++j)
          o[4 + 2 * c + j] = Y::pack(fmaf(16.0f + (float)((hv >> (8 * j)) & 15), vs, vb),
                                     fmaf(16.0f + (float)((hv >> (8 * j + 4)) & 15), vs, vb));
      }
      ok = make_uint4(o[0], o[1], o[2], o[3]);
      ov = make_uint4(o[4], o[5], o[6], o[7]);
    }
    *reinterpret_cast<uint4*>(k + (t0 + tok) * a.k_stride + piece * 8) = ok;
    *reinterpret_cast<uint4*>(v + (t0 + tok) * a.v_stride + piece * 8) = ov;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The checks that both entry points share.  CTI_OK with *empty set: nothing to do.
int check_args(const void* k, const void* v, int dtype, int head_dim, const Args& a,
               int64_t tokens, const void* pages, bool* empty) {
  *empty = false;
  if (a.num_seqs < 0 || tokens < 0 || a.kv_heads <= 0 || a.num_pages < 0 || a.table_cols < 0)
    return CTI_ERR_INVALID_ARG;
  if (dtype != CTI_DTYPE_BF16 && dtype != CTI_DTYPE_F16) return CTI_ERR_UNSUPPORTED;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return CTI_ERR_UNSUPPORTED;
  if (tokens > INT32_MAX - 256 || a.kv_heads > 65535) return CTI_ERR_UNSUPPORTED;
  if (a.num_seqs == 0 || tokens == 0) {
    *empty = true;
    return CTI_OK;
  }
  if (!k || !v || !pages || !a.cu || !a.kv_lens || (!a.table && a.table_cols > 0))
    return CTI_ERR_INVALID_ARG;
  if (!aligned16(k) || !aligned16(v) || !aligned16(pages)) return CTI_ERR_INVALID_ARG;
  const int64_t row = (int64_t)a.kv_heads * head_dim;
  if ((a.k_stride | a.v_stride) % 8 != 0 || a.k_stride < row || a.v_stride < row)
    return CTI_ERR_INVALID_ARG;
  if (a.table_stride < a.table_cols) return CTI_ERR_INVALID_ARG;
  return CTI_OK;
}

template <typename T, int G>
int launch_append(const void* k, const void* v, const Args& a, void* pages, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.tokens + kTokens - 1) / kTokens);
  kv4_append_kernel<T, G><<<grid, kThreads, 0, s>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), a, static_cast<uint8_t*>(pages));
  return cudaGetLastError() == cudaSuccess ? CTI_OK : CTI_ERR_CUDA;
}

template <typename T, int G>
int launch_read(const void* pages, const Args& a, void* k, void* v, cudaStream_t s) {
  const unsigned grid = (unsigned)((a.tokens + kTokens - 1) / kTokens);
  kv4_read_kernel<T, G><<<grid, kThreads, 0, s>>>(static_cast<const uint8_t*>(pages), a,
                                                  static_cast<T*>(k), static_cast<T*>(v));
  return cudaGetLastError() == cudaSuccess ? CTI_OK : CTI_ERR_CUDA;
}

}  // namespace
}  // namespace cti

extern "C" size_t cti_kv4_page_bytes(int kv_heads, int head_dim) {
  if (kv_heads <= 0 || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
  return (size_t)kv_heads * cti::kv4::block_bytes(head_dim / cti::kv4::kGroup);
}

extern "C" int cti_kv4_append(const void* k, const void* v, int64_t k_stride, int64_t v_stride,
                              int dtype, const int32_t* cu_seqlens, const int32_t* kv_lens,
                              const int32_t* page_table, int64_t table_stride, int table_cols,
                              int num_seqs, int64_t tokens, int kv_heads, int head_dim,
                              void* pages, int64_t num_pages, int32_t* status, void* stream) {
  using namespace cti;
  const Args a = {cu_seqlens, kv_lens,   page_table, table_stride, table_cols, num_seqs,
                  (int)tokens, kv_heads, num_pages,  k_stride,     v_stride,   status};
  bool empty;
  const int rc = check_args(k, v, dtype, head_dim, a, tokens, pages, &empty);
  if (rc != CTI_OK || empty) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == CTI_DTYPE_BF16)
    return head_dim == 32   ? launch_append<__nv_bfloat16, 1>(k, v, a, pages, s)
           : head_dim == 64 ? launch_append<__nv_bfloat16, 2>(k, v, a, pages, s)
                            : launch_append<__nv_bfloat16, 4>(k, v, a, pages, s);
  return head_dim == 32   ? launch_append<__half, 1>(k, v, a, pages, s)
         : head_dim == 64 ? launch_append<__half, 2>(k, v, a, pages, s)
                          : launch_append<__half, 4>(k, v, a, pages, s);
}

extern "C" int cti_kv4_read(const void* pages, int64_t num_pages, int dtype,
                            const int32_t* cu_seqlens, const int32_t* kv_lens,
                            const int32_t* page_table, int64_t table_stride, int table_cols,
                            int num_seqs, int64_t tokens, int kv_heads, int head_dim, void* k,
                            void* v, int64_t k_stride, int64_t v_stride, int32_t* status,
                            void* stream) {
  using namespace cti;
  const Args a = {cu_seqlens, kv_lens,   page_table, table_stride, table_cols, num_seqs,
                  (int)tokens, kv_heads, num_pages,  k_stride,     v_stride,   status};
  bool empty;
  const int rc = check_args(k, v, dtype, head_dim, a, tokens, pages, &empty);
  if (rc != CTI_OK || empty) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == CTI_DTYPE_BF16)
    return head_dim == 32   ? launch_read<__nv_bfloat16, 1>(pages, a, k, v, s)
           : head_dim == 64 ? launch_read<__nv_bfloat16, 2>(pages, a, k, v, s)
                            : launch_read<__nv_bfloat16, 4>(pages, a, k, v, s);
  return head_dim == 32   ? launch_read<__half, 1>(pages, a, k, v, s)
         : head_dim == 64 ? launch_read<__half, 2>(pages, a, k, v, s)
                          : launch_read<__half, 4>(pages, a, k, v, s);
}
