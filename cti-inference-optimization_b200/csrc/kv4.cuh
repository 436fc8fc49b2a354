// The 4-bit key/value cache: its format, and what its kernels share.
//
// Groups of 32 consecutive head dims of one token's key (or value) in one
// head are held as 32 codes n in 0..15, a scale s and a base b, both of the
// tensors' 16-bit type T (bf16 or fp16):
//   s = T((max - min) / 15),  b = T(min - 16 s),
//   n = clamp(round((x - b) / s) - 16, 0, 15)   (ties to even; 0 where s = 0)
// and stand for (16 + n) s + b.  The 16 makes a number out of a code without
// arithmetic: a T with the exponent of 16 and the code in its top four
// mantissa bits is 16 + n, so unpacking is a shift and one three-input logic
// operation, and a value is one fused multiply-add away.  b is rounded with
// the 16 s already taken off; that moves the group's grid by half a unit of T in b
// at most.  Where the values lie around zero |b| is about 3 times the largest, so
// this is up to 4 times what the values were rounded by when they became T's; against
// half a step of the codes it is little (values of N(0, 1) in bf16 are held with an
// error of 0.0783, and of 0.0782 with the least value as the base).  A constant group has s = 0 and is held exactly.  A group with
// a value that is not finite, or whose b or 31 s + b in T is not, has s = b =
// NaN: all of it reads back as NaN.  (So every code of a group that has no NaN
// stands for a finite number, and p = 0 leaves out all that is masked.)
//
// A page holds 64 tokens of every KV head; one head's part of it is one
// contiguous block of 2560 G bytes, G = head_dim / 32 groups:
//   K codes 1024 G | K meta 256 G | V codes 1024 G | V meta 256 G
// with the codes in the order in which the attention kernels' matrix
// operands want them.  Token tau = 8 nt + r of the page, group g:
//   K codes  the 32-bit word of dims 32 g + 8 t .. + 7 (t = 0..3) belongs to
//            lane 4 r + t; dims 2 j and 2 j + 1 are the nibbles at bits 4 j
//            and 16 + 4 j.
//   V codes  the 16-bit half of dims 32 g + 4 c .. + 3 (c = 0..7) belongs to
//            lane 4 c + (tau >> 1) % 4, the low half for an even tau, the
//            high one for an odd; dim j is the nibble at bit 4 j.
//   in both, lane l's word i = nt G + g is word i % 4 of its 16-byte vector
//   i / 4, and vector v of lane l is at byte (32 v + l) 16.
//   K meta   [token][g] words: s in the low half, b in the high half.
//   V meta   [token / 2][g] two words: s of both tokens, b of both tokens.
#pragma once

#include "common.cuh"

namespace cti {
namespace kv4 {

constexpr int kSMs = 148;
constexpr int kPage = 64;   // tokens in a page
constexpr int kGroup = 32;  // values that share a scale and a base

// Bytes of one head's part of a page, and where its sections start.
__host__ __device__ constexpr int block_bytes(int G) { return 2560 * G; }
__host__ __device__ constexpr int part_bytes(int G) { return 1280 * G; }  // of keys, or values
__host__ __device__ constexpr int k_meta_at(int G) { return 1024 * G; }
__host__ __device__ constexpr int v_codes_at(int G) { return 1280 * G; }
__host__ __device__ constexpr int v_meta_at(int G) { return 2304 * G; }

// Byte of lane `lane`'s code word i inside a codes section.
CTI_DEVICE int code_word_at(int i, int lane) { return ((i >> 2) * 32 + lane) * 16 + (i & 3) * 4; }
CTI_DEVICE int k_word_at(int tau, int g, int t, int G) {
  return code_word_at((tau >> 3) * G + g, (tau & 7) * 4 + t);
}
CTI_DEVICE int v_half_at(int tau, int g, int c, int G) {
  return code_word_at((tau >> 3) * G + g, c * 4 + ((tau >> 1) & 3)) + (tau & 1) * 2;
}
CTI_DEVICE int k_meta_word_at(int tau, int g, int G) { return (tau * G + g) * 4; }
CTI_DEVICE int v_meta_half_at(int tau, int g, int G) {  // s; b is 4 bytes further
  return ((tau >> 1) * G + g) * 8 + (tau & 1) * 2;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The two 16-bit types.
template <typename T>
struct Type16;
template <>
struct Type16<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x41804180u;  // 16.0 twice; the code goes to bits 3..6
  static constexpr int kShift = 3;
  static constexpr uint32_t kTopBits = 0xffff0000u;  // of a float, that T holds exactly
  CTI_DEVICE static float to_float(uint32_t h) { return __uint_as_float(h << 16); }
  CTI_DEVICE static float low(uint32_t w) { return __uint_as_float(w << 16); }
  CTI_DEVICE static float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
  CTI_DEVICE static uint32_t bits(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
  CTI_DEVICE static uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct Type16<__half> {
  static constexpr uint32_t kMagic = 0x4c004c00u;  // 16.0 twice; the code goes to bits 6..9
  static constexpr int kShift = 6;
  static constexpr uint32_t kTopBits = 0xffffe000u;  // in T's normal range
  CTI_DEVICE static float to_float(uint32_t h) {
    return __half2float(__ushort_as_half((unsigned short)h));
  }
  CTI_DEVICE static float low(uint32_t w) { return to_float(w & 0xffffu); }
  CTI_DEVICE static float high(uint32_t w) { return to_float(w >> 16); }
  CTI_DEVICE static uint32_t bits(float f) { return __half_as_ushort(__float2half_rn(f)); }
  CTI_DEVICE static uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
};

// a b + c of both halves in T, rounded once.
template <typename T>
CTI_DEVICE uint32_t fma2(uint32_t a, uint32_t b, uint32_t c);
template <>
CTI_DEVICE uint32_t fma2<__nv_bfloat16>(uint32_t a, uint32_t b, uint32_t c) {
  __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&a),
                             *reinterpret_cast<__nv_bfloat162*>(&b),
                             *reinterpret_cast<__nv_bfloat162*>(&c));
  return *reinterpret_cast<uint32_t*>(&r);
}
template <>
CTI_DEVICE uint32_t fma2<__half>(uint32_t a, uint32_t b, uint32_t c) {
  __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b),
                      *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<uint32_t*>(&r);
}

// 16 + n twice from nibble j of both halves of a word.
template <typename T>
CTI_DEVICE uint32_t code_pair(uint32_t w, int j) {
  constexpr int s = Type16<T>::kShift;
  const int r = 4 * j - s;  // right shift that brings the nibble to bits s..s+3
  const uint32_t x = r < 0 ? w << -r : w >> r;
  return (x & (0x000f000fu << s)) | Type16<T>::kMagic;
}

// Largest s in [0, n) with cu[s] <= t (cu[0] <= t < cu[n]).
CTI_DEVICE int sequence_of(const int32_t* __restrict__ cu, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The page of position p of sequence s, or -1.
CTI_DEVICE int64_t page_of(const int32_t* __restrict__ table, int64_t table_stride, int table_cols,
                           int64_t num_pages, int s, int64_t p, int32_t* status) {
  if (p >= 0 && p / kPage < table_cols) {
    const int64_t page = __ldg(table + s * table_stride + p / kPage);
    if (page >= 0 && page < num_pages) return page;
  }
  raise_status(status, CTI_ERR_BOUNDS, s);
  return -1;
}

}  // namespace kv4
}  // namespace cti
