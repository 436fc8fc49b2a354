// Writing tokens into the 4-bit key/value cache and reading them back
// (format: kv4.cuh).
//
// A block takes packed tokens side by side, 32 / G of them (G = head_dim / 32)
// or a multiple.  In a page, 16 bytes hold a word each of G groups in 4 / G
// octets of tokens.  A warp's lanes take those four words; with them a token's
// two halves of the group (append; 16 dims to a lane) or four quarters (read);
// and 4 or 2 tokens side by side, whose values share sectors.  So whole sectors
// move where tokens follow each other in a page, and nothing is lost where each is
// of its own sequence.  (With a token's groups side by side in a warp instead,
// sectors are written in pieces: 38 us for 25 to append 24,576 tokens of 8 heads
// of 64, in L2.)
// Either way moves 4 + 1.25 bytes per pair of a key's and a value's element.
// Measured, 278,000 tokens of 8 heads of 32: 113 us to append (51 % of the copy
// bandwidth) and 79 us to read back (73 %).  Bound by latency: warps wait for loads
// first (3.7 cycles an instruction when appending, 5.9 when reading), with 28 and 40 of
// 64 warps there and 58 and 64 % of the issue slots taken; 17 instructions for 32
// values of a warp are what appending cannot hide it with.
#include <cfloat>

#include "kv4.cuh"

namespace cti {
namespace {

using namespace kv4;

constexpr int kThreads = 256;
constexpr int kTokens = 128;  // packed tokens of a block, at most
constexpr int64_t kMaxStride = ((int64_t)1 << 31) / kTokens;

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
  int tile;  // packed tokens of a block
};

CTI_DEVICE float min3_nan(float a, float b, float c) {
  float d;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
CTI_DEVICE float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The smaller of both halves of two numbers of T; NaN if one is.
template <typename T>
CTI_DEVICE uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (Type16<T>::kShift == 3)
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Codes are exact, whatever fp32 rounds.  With a = x - b, the quotient a / s
// is rounded to nearest by one correction of its estimate's remainder
// (Markstein), and then to a whole number, ties to even, by adding 1.5 2^23,
// which leaves k = 16 + n in the low bits.  Rounding twice is right: a has 24
// bits and lies in [16 s, 32 s), so a / s is either a border k + 1/2 itself
// or at least 2^-19 away from it, one unit of the quotient.  Two cases are
// looked at again, out of line:
//   - an end of the group comes out below code 0 or above 15, because b's or
//     s's rounding moved the grid;
//   - a was rounded onto a border that x - b does not lie on.  That takes an |x|
//     below 2^-13 |b| (fp16; bf16: 2^-16), so -b is that close to the border, which is
//     2^-8 s at most; x's side decides.  (In bf16 borders are multiples of 2^-13 of
//     b's binade away from -b, too far, unless -b lies on one itself.)
constexpr float kRound = 12582912.0f;  // 1.5 2^23
constexpr uint32_t kRoundBits = 0x4b400000u;

enum Order { kKeys, kValues };  // dims 2 j at 4 j, 2 j + 1 at 16 + 4 j; or dim j at 4 j
__host__ __device__ constexpr int dim_at(Order order, int nibble) {
  return order == kValues ? nibble : nibble < 4 ? 2 * nibble : 2 * nibble - 7;
}

template <typename T>
CTI_DEVICE void unpack(const uint4& raw, float* x) {
  using Y = Type16<T>;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Y::low(w[i]);
    x[2 * i + 1] = Y::high(w[i]);
  }
}

// The nibbles of the 8 t (kRoundBits + 16 + n as bits): a chain of shift-adds
// less what is not n.
template <Order ORDER>
CTI_DEVICE uint32_t pack_codes(const float* t) {
  uint32_t word = 0, less = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) {
    word = word * 16 + __float_as_uint(t[dim_at(ORDER, i)]);
    less = less * 16 + kRoundBits + 16;
  }
  return word - less;
}

// The cases above, one value at a time: k is at most one off, the remainder
// r = a - k s is exact, and where it reaches s / 2 the rounding error of a
// decides.
template <typename T, Order ORDER>
__device__ __noinline__ uint32_t codes_again(uint4 raw, float s, float b, float inv) {
  float x[8], t[8];
  unpack<T>(raw, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i] - b, z = a - x[i];
    const float err = (x[i] - (a - z)) + (-b - z);  // x - b = a + err
    float k = rintf(a * inv);
    const float r = fmaf(-s, k, a);
    const float over = (fabsf(r) - 0.5f * s) + (r > 0.0f ? err : -err);
    if (fabsf(r) >= 0.5f * s && (over > 0.0f || (over == 0.0f && ((int)k & 1) != 0)))
      k += r > 0.0f ? 1.0f : -1.0f;
    t[i] = kRound + fminf(fmaxf(k, 16.0f), 31.0f);
  }
  return pack_codes<ORDER>(t);
}

// Packs 16 values of a group of 32 (the lane whose number differs in bit 0 has
// the others) into two words of codes.  Also the group's scale and base, 16
// bits each.  Bound by instructions: about 9 a value with the group's part, the
// values' arithmetic two at a time.  (With 8 values a lane, where the group's
// part is done by four lanes: 13.)
template <typename T, Order ORDER>
CTI_DEVICE void quantise(const uint4 (&raw)[2], uint32_t (&word)[2], uint32_t& s_bits,
                         uint32_t& b_bits) {
  using Y = Type16<T>;
  float x[16];
  unpack<T>(raw[0], x);
  unpack<T>(raw[1], x + 8);
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 15; i += 2) {
    lo = min3_nan(lo, x[i], x[i + 1]);
    hi = max3_nan(hi, x[i], x[i + 1]);
  }
  lo = min3_nan(lo, x[15], x[15]);
  hi = max3_nan(hi, x[15], x[15]);
  // Both ends in one exchange: they are numbers of T.
  uint32_t both = Y::pack(lo, -hi);
  both = min2_nan<T>(both, __shfl_xor_sync(0xffffffffu, both, 1));
  lo = Y::low(both);
  hi = -Y::high(both);
  // (hi - lo) / 15 in the same way as the codes' quotients; its rounding on to
  // T is right too: it is nearer to the true value than to any border of T that
  // it does not lie on.
  const float range = hi - lo;
  const float q = range * (1.0f / 15.0f);
  s_bits = Y::bits(fmaf(fmaf(-15.0f, q, range), 1.0f / 15.0f, q));
  const float s = Y::to_float(s_bits);
  b_bits = Y::bits(fmaf(-16.0f, s, lo));
  const float b = Y::to_float(b_bits);
  const float top = Y::to_float(Y::bits(fmaf(31.0f, s, b)));  // what the last code stands for
  if (!(s >= FLT_MIN && s <= FLT_MAX && fabsf(b) <= FLT_MAX && top <= FLT_MAX)) {
    word[0] = word[1] = 0;
    if (s < FLT_MIN) {  // below the smallest normal fp32 number: a constant group
      s_bits = 0;
      b_bits = Y::bits(lo);
    } else {
      s_bits = b_bits = 0x7fffu;  // NaN in both types
    }
    return;
  }
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  // a / s for two values at once
  const uint64_t ns2 = f2_pack(-s, -s), nb2 = f2_pack(-b, -b), inv2 = f2_pack(inv, inv);
  const uint64_t add2 = f2_pack(kRound, kRound);
  auto quotient = [&](float x0, float x1) {
    const uint64_t a = f2_add(f2_pack(x0, x1), nb2);
    const uint64_t e = f2_mul(a, inv2);
    return f2_fma(f2_fma(ns2, e, a), inv2, e);
  };
  float t_lo, t_hi;
  f2_unpack(f2_add(quotient(lo, hi), add2), t_lo, t_hi);
  bool again = t_lo < kRound + 16.0f || t_hi > kRound + 31.0f;
  // -b next to a border: -b / s next to a whole number and a half
  constexpr float kNear = Y::kShift == 3 ? 0.0f : 0x1.01p-8f;
  const float e0 = -b * inv, e1 = fmaf(fmaf(-s, e0, -b), inv, e0);
  if (0.5f - fabsf(e1 - ((e1 + kRound) - kRound)) <= kNear) {
    float least = INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) least = fminf(least, x[i] == 0.0f ? INFINITY : fabsf(x[i]));
    again = again || least < fabsf(b) * 0x1p-12f;
  }
  if (again) {
    word[0] = codes_again<T, ORDER>(raw[0], s, b, inv);
    word[1] = codes_again<T, ORDER>(raw[1], s, b, inv);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      f2_unpack(f2_add(quotient(x[8 * h + i], x[8 * h + i + 1]), add2), t[i], t[i + 1]);
    word[h] = pack_codes<ORDER>(t);
  }
}

// What a K word stands for in T.
template <typename T>
CTI_DEVICE uint4 k_values(uint32_t w, uint32_t meta) {
  const uint32_t s = __byte_perm(meta, 0, 0x1010), b = __byte_perm(meta, 0, 0x3232);
  return make_uint4(fma2<T>(code_pair<T>(w, 0), s, b), fma2<T>(code_pair<T>(w, 1), s, b),
                    fma2<T>(code_pair<T>(w, 2), s, b), fma2<T>(code_pair<T>(w, 3), s, b));
}
// What a V word stands for: its even token's 4 values, and its odd one's.
template <typename T>
CTI_DEVICE void v_values(uint32_t w, uint32_t s, uint32_t b, uint2& even, uint2& odd) {
  uint32_t x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = fma2<T>(code_pair<T>(w, j), s, b);
  even = make_uint2(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410));
  odd = make_uint2(__byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
}

// Where a packed token's key and value live.
struct Place {
  int64_t page;  // its offset in bytes; -1: nowhere (an index outside its buffer; the
                 // status word says so); -2: a token of no sequence
  int slot;
};

// The places of the block's a.tile packed tokens from t0 on.  All threads of the
// block.
template <int G>
CTI_DEVICE void find_places(const Args& a, int t0, Place (&places)[kTokens]) {
  static_assert(kTokens <= kThreads, "a thread per token");
  const int lane = lane_id(), first = t0 + warp_id() * 32, t = first + lane;
  if (warp_id() * 32 < a.tile) {
    Place at = {-2, 0};
    const bool live = warp_id() * 32 + lane < a.tile && t < a.tokens && t >= __ldg(a.cu) &&
                      t < __ldg(a.cu + a.num_seqs);
    // As many tokens in each sequence: no search.
    int s = live ? (int)((int64_t)t * a.num_seqs / a.tokens) : 0;
    if (!__all_sync(0xffffffffu, !live || (__ldg(a.cu + s) <= t && t < __ldg(a.cu + s + 1)))) {
      // The sequence of the warp's first token, 32 borders at a time; the others'
      // are found among the next 32.
      int lo = 0, hi = a.num_seqs;  // cu[lo] <= first (or lo = 0), and first < cu[hi]
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, border = lo + (lane + 1) * step;
        const uint32_t le =
            __ballot_sync(0xffffffffu, border < hi && __ldg(a.cu + border) <= first);
        const int last = __popc(le);
        hi = min(hi, lo + (last + 1) * step);
        lo += last * step;
      }
      const int end = __ldg(a.cu + min(lo + 1 + lane, a.num_seqs));
      int past = 0;
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (__shfl_sync(0xffffffffu, end, past + step - 1) <= t) past += step;
      const bool beyond = __shfl_sync(0xffffffffu, end, 31) <= t;  // empty sequences between
      if (live) s = beyond ? sequence_of(a.cu, a.num_seqs, t) : lo + past;
    }
    if (live) {
      const int64_t p = (int64_t)__ldg(a.kv_lens + s) - __ldg(a.cu + s + 1) + t;
      const int64_t page =
          page_of(a.table, a.table_stride, a.table_cols, a.num_pages, s, p, a.status);
      at.page = page < 0 ? -1 : page * a.kv_heads * block_bytes(G);
      at.slot = (int)(p & (kPage - 1));
    }
    if (warp_id() * 32 + lane < a.tile) places[warp_id() * 32 + lane] = at;
  }
  __syncthreads();
}

// What a warp does, turn by turn, and its lanes' parts in it: PARTS lanes share a
// group of a token.
template <int G, int PARTS>
struct Turns {
  static constexpr int kUnit = 32 / G;            // tokens of 4 / G octets,
  static constexpr int kSteps = PARTS;            // which take so many turns in one head
  static constexpr int kSide = 32 / (4 * PARTS);  // tokens of an octet in a turn
  static constexpr int kWarps = kThreads / 32;
  int head, tok, end;  // of the tokens, where the turns end
  int heads;
  CTI_DEVICE Turns(int tile, int heads_) : heads(heads_) {
    const int lane = lane_id(), warp = warp_id();
    head = warp / kSteps;
    end = heads > 0 ? tile : 0;
    tok = (lane / PARTS & 3) / G * 8 + warp % kSteps * kSide + lane / (4 * PARTS);
    wrap();
  }
  CTI_DEVICE void wrap() {
    while (head >= heads && tok < end) head -= heads, tok += kUnit;
  }
  CTI_DEVICE void next() {
    head += kWarps / kSteps;
    wrap();
  }
  // The same for a whole warp: its tokens are all of one unit.
  CTI_DEVICE bool more() const { return tok < end; }
  CTI_DEVICE static int group() { return (lane_id() / PARTS & 3) % G; }
  CTI_DEVICE static int part() { return lane_id() % PARTS; }
};

// The heads of this block: gridDim.y blocks share a tile.
CTI_DEVICE int2 heads_of(const Args& a) {
  const int per = (a.kv_heads + gridDim.y - 1) / gridDim.y;
  const int first = min(a.kv_heads, per * (int)blockIdx.y);
  return make_int2(first, min(a.kv_heads - first, per));
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads)
    kv4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, Args a,
                      uint8_t* __restrict__ pages) {
  using Turn = Turns<G, 2>;
  __shared__ Place places[kTokens];
  const int t0 = blockIdx.x * a.tile;
  find_places<G>(a, t0, places);
  const int2 heads = heads_of(a);
  // Offsets of 32 bits: the tile's tokens are within 2^31 elements of each other.
  const T* kt = k + t0 * a.k_stride;
  const T* vt = v + t0 * a.v_stride;
  const int g = Turn::group(), part = Turn::part();
  for (Turn i(a.tile, heads.y); i.more(); i.next()) {
    const Place at = places[i.tok];
    const int head = heads.x + i.head, piece = (2 * (head * G + g) + part) * 16;
    uint4 rk[2], rv[2];
    rk[0] = rk[1] = rv[0] = rv[1] = make_uint4(0, 0, 0, 0);
    if (at.page >= 0) {
      const uint4* pk = reinterpret_cast<const uint4*>(kt + (i.tok * (int)a.k_stride + piece));
      const uint4* pv = reinterpret_cast<const uint4*>(vt + (i.tok * (int)a.v_stride + piece));
      rk[0] = __ldg(pk);
      rk[1] = __ldg(pk + 1);
      rv[0] = __ldg(pv);
      rv[1] = __ldg(pv + 1);
    }
    uint32_t ks, kb, vs, vb, wk[2], wv[2];
    quantise<T, kKeys>(rk, wk, ks, kb);
    quantise<T, kValues>(rv, wv, vs, vb);
    if (at.page < 0) continue;  // the loop's end is the same for a whole warp
    uint8_t* block = pages + at.page + head * block_bytes(G);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      *reinterpret_cast<uint32_t*>(block + k_word_at(at.slot, g, 2 * part + x, G)) = wk[x];
#pragma unroll
      for (int c = 0; c < 2; ++c)
        *reinterpret_cast<uint16_t*>(block + v_codes_at(G) +
                                     v_half_at(at.slot, g, 4 * part + 2 * x + c, G)) =
            (uint16_t)(wv[x] >> (16 * c));
    }
    if (part == 0) {
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
  using Turn = Turns<G, 4>;
  __shared__ Place places[kTokens];
  const int t0 = blockIdx.x * a.tile;
  grid_dependency_wait();
  find_places<G>(a, t0, places);
  const int2 heads = heads_of(a);
  T* kt = k + t0 * a.k_stride;
  T* vt = v + t0 * a.v_stride;
  const int g = Turn::group(), part = Turn::part();
  constexpr int N = 2;  // turns at once: all loads first
  for (Turn i(a.tile, heads.y); i.more();) {
    uint32_t wk[N], mk[N], h0[N], h1[N];
    uint2 mv[N];
    int64_t page[N];
    int tok[N], piece[N];
    bool odd[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      page[n] = -2;
      if (!i.more()) continue;
      const Place at = places[i.tok];
      const int head = heads.x + i.head;
      page[n] = at.page;
      tok[n] = i.tok;
      piece[n] = (4 * (head * G + g) + part) * 8;
      odd[n] = at.slot & 1;
      i.next();
      if (at.page < 0) continue;
      const uint8_t* block = pages + at.page + head * block_bytes(G);
      wk[n] = __ldg(reinterpret_cast<const uint32_t*>(block + k_word_at(at.slot, g, part, G)));
      mk[n] = __ldg(reinterpret_cast<const uint32_t*>(block + k_meta_at(G) +
                                                      k_meta_word_at(at.slot, g, G)));
      mv[n] = __ldg(reinterpret_cast<const uint2*>(block + v_meta_at(G) +
                                                   v_meta_half_at(at.slot & ~1, g, G)));
      const uint8_t* vc = block + v_codes_at(G);
      h0[n] = __ldg(reinterpret_cast<const uint16_t*>(vc + v_half_at(at.slot, g, 2 * part, G)));
      h1[n] = __ldg(reinterpret_cast<const uint16_t*>(vc + v_half_at(at.slot, g, 2 * part + 1, G)));
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (page[n] == -2) continue;
      uint4 ok = make_uint4(0, 0, 0, 0), ov = ok;
      if (page[n] >= 0) {
        const uint32_t both = odd[n] ? 0x3232 : 0x1010;
        uint2 v0, v1;
        v_values<T>(h0[n] | h1[n] << 16, __byte_perm(mv[n].x, 0, both),
                    __byte_perm(mv[n].y, 0, both), v0, v1);
        ok = k_values<T>(wk[n], mk[n]);
        ov = make_uint4(v0.x, v0.y, v1.x, v1.y);
      }
      *reinterpret_cast<uint4*>(kt + (tok[n] * (int)a.k_stride + piece[n])) = ok;
      *reinterpret_cast<uint4*>(vt + (tok[n] * (int)a.v_stride + piece[n])) = ov;
    }
  }
}

// The checks that both entry points share.  CTI_OK with *empty set: nothing to do.
int check_args(const void* k, const void* v, int dtype, int head_dim, const Args& a,
               int64_t tokens, const void* pages, bool* empty) {
  *empty = false;
  if (a.num_seqs < 0 || tokens < 0 || a.kv_heads <= 0 || a.num_pages < 0 || a.table_cols < 0)
    return CTI_ERR_INVALID_ARG;
  if (dtype != CTI_DTYPE_BF16 && dtype != CTI_DTYPE_F16) return CTI_ERR_UNSUPPORTED;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128) return CTI_ERR_UNSUPPORTED;
  if (tokens > INT32_MAX - 256 || a.num_seqs > INT32_MAX - 256 || a.kv_heads > 65535)
    return CTI_ERR_UNSUPPORTED;
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
  // A tile's tokens are within 2^31 elements of each other.
  if (a.k_stride > kMaxStride || a.v_stride > kMaxStride) return CTI_ERR_UNSUPPORTED;
  if (a.table_stride < a.table_cols) return CTI_ERR_INVALID_ARG;
  return CTI_OK;
}

// The tokens of a block and the grid of a call: a turn for each warp; blocks that
// share a tile by heads, until there are four blocks for each SM; and two tiles'
// tokens to a block where that leaves 8 for each SM (278,000 tokens of 8 heads of 32:
// 125 us become 115 to append, 92 become 82 to read; four: 113 and 84).
dim3 plan(Args& a, int G) {
  const int heads = kThreads / 64;  // that keep a block's warps busy
  a.tile = 32 / G * (a.kv_heads >= heads ? 1 : (heads + a.kv_heads - 1) / a.kv_heads);
  if (a.tile < kTokens && a.tokens >= (int64_t)a.tile * 2 * 8 * kSMs) a.tile *= 2;
  const int64_t tiles = ((int64_t)a.tokens + a.tile - 1) / a.tile;
  const int64_t share = (kSMs * 4 + tiles - 1) / tiles;
  const int64_t most = (a.kv_heads + heads - 1) / heads;
  return dim3((unsigned)tiles, (unsigned)(share < most ? share : most));
}

template <typename T, int G>
int launch_append(const void* k, const void* v, Args a, void* pages, cudaStream_t s) {
  const dim3 grid = plan(a, G);
  kv4_append_kernel<T, G><<<grid, kThreads, 0, s>>>(
      static_cast<const T*>(k), static_cast<const T*>(v), a, static_cast<uint8_t*>(pages));
  return cudaGetLastError() == cudaSuccess ? CTI_OK : CTI_ERR_CUDA;
}

template <typename T, int G>
int launch_read(const void* pages, Args a, void* k, void* v, cudaStream_t s) {
  const dim3 grid = plan(a, G);
  return launch_dependent(kv4_read_kernel<T, G>, grid, dim3(kThreads), 0, s,
                          static_cast<const uint8_t*>(pages), a, static_cast<T*>(k),
                          static_cast<T*>(v)) == cudaSuccess
             ? CTI_OK
             : CTI_ERR_CUDA;
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
                  (int)tokens, kv_heads, num_pages,  k_stride,     v_stride,   status,   0};
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
                  (int)tokens, kv_heads, num_pages,  k_stride,     v_stride,   status,   0};
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
