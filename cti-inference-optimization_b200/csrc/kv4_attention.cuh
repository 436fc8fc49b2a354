// What the kernels of the attention over the 4-bit cache share: their
// arguments, and how far a row's exponent offset may lag.
#pragma once

#include "kv4.cuh"

namespace cti {
namespace kv4 {

// A row's exponent offset m is only raised (and O, l rescaled) when a score
// exceeds it by this power of 2: p <= 2^kSlack.
constexpr float kSlack = 8.0f;
// Exponent that weights of 1 are formed with where P is fp16: 2^kSlack of it are
// within fp16, and small weights have the most bits.
constexpr float kPUnitFp16 = 7.0f;

// x / d for 0 <= x < 2^31 by a multiplication and a shift (the round-up
// method of Granlund and Montgomery).
struct Divisor {
  uint32_t mul, shift;
  explicit Divisor(uint32_t d) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  CTI_DEVICE uint32_t operator()(uint32_t x) const { return (__umulhi(mul, x) + x) >> shift; }
};

struct Args {
  const int32_t* cu;
  const int32_t* kv_lens;
  const int32_t* table;
  int64_t table_stride;
  int table_cols;
  int num_seqs;
  int tokens;
  int heads, kv_heads, group;
  float scale_m;     // |scale| log2(e) = scale_m 2^scale_e
  int scale_e;
  float sign;        // of scale, which goes to the queries: 1, -1, or 0
  int causal;
  int64_t num_pages;
  int64_t q_stride;
  Divisor by_group, by_kv_heads;
  int shared;          // a block's warps share a row tile; else each has its own
  int chunk;           // pages of a sequence for a block (gridDim.z > 1)
  float* ws_o;         // [splits][tokens * heads][D], O / l; splits > 1 only
  float2* ws_ml;       // [splits][tokens * heads], m and l
  int32_t* status;
};

// 2^e, for -126 <= e <= 127; infinity for 128.
CTI_DEVICE float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The exponent k that queries of at most `most` are scaled by, to 2^14 .. 2^15 in fp16.  Where
// |scale| 2^-k would leave fp32's normal numbers they stay smaller: a rounding in fp16 is
// nothing then, even to keys of 2^127.
CTI_DEVICE int query_exponent(float most, const Args& a) {
  const int k = 14 + 127 - (int)(__float_as_uint(most) >> 23);
  return most * fabsf(a.sign) > 0.0f ? max(-113, min(k, min(100, a.scale_e + 126))) : 0;
}

// A sequence whose offsets lie outside the tokens, or fall, is refused.  Where
// sequences are split, its rows' l of the first split says so to the join (-1;
// no other l is negative), which leaves them as they were.  One block of a
// sequence's KV head calls this.
static __device__ __noinline__ void refuse_rows(float2* ws_ml, int begin, int end, int heads,
                                                int group, int kvh) {
#pragma unroll 1
  for (int t = begin + (int)threadIdx.x; t < end; t += blockDim.x)
#pragma unroll 1
    for (int h = 0; h < group; ++h)
      ws_ml[(int64_t)t * heads + kvh * group + h] = make_float2(-INFINITY, -1.0f);
}

CTI_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

CTI_DEVICE float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Exponent bits of T: set in infinities and NaN.
template <typename T>
struct Inf16;
template <>
struct Inf16<__nv_bfloat16> {
  static constexpr uint32_t kBits = 0x7f80u;
};
template <>
struct Inf16<__half> {
  static constexpr uint32_t kBits = 0x7c00u;
};

// Rows tiles of 128 on the tensor cores (kv4_tiles.cu).  tiles: 128-row tiles
// that a block takes side by side, 1 or 2; y: of a sequence; splits: as for
// the row kernel.  CTI_OK or a CTI_ERR code.
int launch_tiles(const void* q, const void* pages, const Args& a, int dtype, int head_dim,
                 int tiles, int64_t y, int splits, void* out, cudaStream_t s);

}  // namespace kv4
}  // namespace cti
