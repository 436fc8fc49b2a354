// Writing tokens into the 4-bit key/value cache and reading them back
// (format: kv4.cuh).
//
// Two ways, by the tokens that a sequence has in the call:
//   runs    a block finds the runs (tokens side by side in one page) that start
//           among 64 or 128 packed tokens; a warp takes a run's keys or values
//           in one head, with lanes laid out as the page's, so that it moves
//           whole sectors of codes.
//   tokens  a block takes 8 packed tokens, every thread 16 dims of a token's
//           key and value.  For calls with a few tokens per sequence, whose
//           runs would leave most lanes of a warp idle.
// Either way moves 4 + 1.25 bytes per pair of a key's and a value's element.
// Measured, 278,000 tokens of 8 heads of 32: 123 us to append (bound by
// instructions, 17 for 32 values of a warp; 47 % of the copy bandwidth) and 75
// us to read back (latency; 76 %).
#include <cfloat>

#include "kv4.cuh"

namespace cti {
namespace {

using namespace kv4;

constexpr int kSMs = 148;
constexpr int kThreads = 256;
constexpr int kTokens = 8;      // packed tokens of a block, by tokens
constexpr int kRunTokens = 128;  // and by runs, at most
constexpr int64_t kMaxStride = (int64_t)1 << 24;
// A sequence's tokens in a call, on average, from which runs are used.
constexpr int kRunsFrom = 8;

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
//   - a was rounded, which takes an |x| far below |b|, where a is -b, and -b
//     lies on a border: then x's sign decides.
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
  if (!(s >= FLT_MIN && s <= FLT_MAX && fabsf(b) <= FLT_MAX)) {
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
  // -b on a border: -b / s = a whole number and a half
  const float e0 = -b * inv, e1 = fmaf(fmaf(-s, e0, -b), inv, e0);
  if (fabsf(e1 - ((e1 + kRound) - kRound)) == 0.5f) {
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

CTI_DEVICE uint32_t twice(uint32_t h) { return __byte_perm(h, h, 0x1010); }

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

// Place of packed token t, page -2 where it is of no sequence.
CTI_DEVICE Place find_place(const Args& a, int t) {
  Place at = {-2, 0};
  if (t < a.tokens && t >= __ldg(a.cu) && t < __ldg(a.cu + a.num_seqs))
    at = place_of(a.cu, a.kv_lens, a.table, a.table_stride, a.table_cols, a.num_seqs, a.tokens,
                  a.num_pages, t, a.status);
  return at;
}

// ---------------------------------------------------------------------------
// By tokens.
// ---------------------------------------------------------------------------
template <typename T, int G>
__global__ void __launch_bounds__(kThreads)
    kv4_append_tokens_kernel(const T* __restrict__ k, const T* __restrict__ v, Args a,
                             uint8_t* __restrict__ pages) {
  __shared__ Place places[kTokens];
  const int t0 = blockIdx.x * kTokens;
  if (threadIdx.x < kTokens) places[threadIdx.x] = find_place(a, t0 + threadIdx.x);
  __syncthreads();
  const int per = a.kv_heads * G * 2;  // 16-dim pieces of a token
  const int total = (kTokens * per + 31) & ~31;
  for (int i = threadIdx.x; i < total; i += kThreads) {
    const int tok = i / per, piece = i - tok * per;
    const Place at = tok < kTokens ? places[tok] : Place{-1, 0};
    const int head = piece / (2 * G), g = (piece >> 1) & (G - 1), t = 2 * (piece & 1);
    const bool live = at.page >= 0;
    uint4 rk[2], rv[2];
    rk[0] = rk[1] = rv[0] = rv[1] = make_uint4(0, 0, 0, 0);
    if (live) {
      const uint4* pk =
          reinterpret_cast<const uint4*>(k + (t0 + tok) * a.k_stride + piece * 16);
      const uint4* pv =
          reinterpret_cast<const uint4*>(v + (t0 + tok) * a.v_stride + piece * 16);
      rk[0] = __ldg(pk);
      rk[1] = __ldg(pk + 1);
      rv[0] = __ldg(pv);
      rv[1] = __ldg(pv + 1);
    }
    uint32_t ks, kb, vs, vb, wk[2], wv[2];
    quantise<T, kKeys>(rk, wk, ks, kb);
    quantise<T, kValues>(rv, wv, vs, vb);
    if (!live) continue;  // the loop's bound is the same for a whole warp
    uint8_t* block = pages + (at.page * a.kv_heads + head) * (int64_t)block_bytes(G);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      *reinterpret_cast<uint32_t*>(block + k_word_at(at.slot, g, t + x, G)) = wk[x];
#pragma unroll
      for (int c = 0; c < 2; ++c)
        *reinterpret_cast<uint16_t*>(block + v_codes_at(G) +
                                     v_half_at(at.slot, g, 2 * (t + x) + c, G)) =
            (uint16_t)(wv[x] >> (16 * c));
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
    kv4_read_tokens_kernel(const uint8_t* __restrict__ pages, Args a, T* __restrict__ k,
                           T* __restrict__ v) {
  __shared__ Place places[kTokens];
  const int t0 = blockIdx.x * kTokens;
  grid_dependency_wait();
  if (threadIdx.x < kTokens) places[threadIdx.x] = find_place(a, t0 + threadIdx.x);
  __syncthreads();
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
      const uint32_t wk =
          __ldg(reinterpret_cast<const uint32_t*>(block + k_word_at(at.slot, g, t, G)));
      const uint32_t mk = __ldg(
          reinterpret_cast<const uint32_t*>(block + k_meta_at(G) + k_meta_word_at(at.slot, g, G)));
      const uint8_t* vm = block + v_meta_at(G) + v_meta_half_at(at.slot, g, G);
      const uint32_t vs = __ldg(reinterpret_cast<const uint16_t*>(vm));
      const uint32_t vb = __ldg(reinterpret_cast<const uint16_t*>(vm + 4));
      const uint8_t* vc = block + v_codes_at(G);
      const uint32_t h0 =
          __ldg(reinterpret_cast<const uint16_t*>(vc + v_half_at(at.slot, g, 2 * t, G)));
      const uint32_t h1 =
          __ldg(reinterpret_cast<const uint16_t*>(vc + v_half_at(at.slot, g, 2 * t + 1, G)));
      uint2 v0, v1;
      v_values<T>(h0 | h1 << 16, twice(vs), twice(vb), v0, v1);
      ok = k_values<T>(wk, mk);
      ov = make_uint4(v0.x, v0.y, v1.x, v1.y);
    }
    *reinterpret_cast<uint4*>(k + (t0 + tok) * a.k_stride + piece * 8) = ok;
    *reinterpret_cast<uint4*>(v + (t0 + tok) * a.v_stride + piece * 8) = ov;
  }
}

// ---------------------------------------------------------------------------
// By runs.
// ---------------------------------------------------------------------------
// Side by side in one page: packed tokens [start, start + count), from `slot`
// of the page on.
struct Run {
  int64_t page;
  int start, count, slot;
};

// The runs that START among the block's a.tile packed tokens from t0 on, so
// that no run is cut at a tile's end.  All threads of the block; returns their
// number.
CTI_DEVICE int find_runs(const Args& a, int t0, Run (&runs)[kRunTokens]) {
  static_assert(kRunTokens % 32 == 0 && kRunTokens <= kThreads, "a thread per token");
  __shared__ int32_t ends[kRunTokens];  // cu[s0 + 1 + i]
  __shared__ uint32_t starts[kRunTokens / 32];
  __shared__ int s0_shared;
  const int i = threadIdx.x, tile = a.tile;
  if (i < 32) {  // the sequence of token t0, 32 borders at a time
    int lo = 0, hi = a.num_seqs;  // cu[lo] <= t0 (or lo = 0), and t0 < cu[hi]
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, at = lo + (i + 1) * step;
      const uint32_t le = __ballot_sync(0xffffffffu, at < hi && __ldg(a.cu + at) <= t0);
      const int last = __popc(le);
      hi = min(hi, lo + (last + 1) * step);
      lo += last * step;
    }
    if (i == 0) s0_shared = lo;
  }
  __syncthreads();
  const int s0 = s0_shared;
  if (i < tile) ends[i] = __ldg(a.cu + min(s0 + 1 + i, a.num_seqs));
  __syncthreads();
  const int t = t0 + i;
  Run run = {-2, t, 0, 0};
  if (i < tile && t < a.tokens && t >= __ldg(a.cu) && t < __ldg(a.cu + a.num_seqs)) {
    int s = s0;
    if (ends[tile - 1] > t) {
      int lo = -1, hi = tile - 1;  // ends[lo] <= t < ends[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] <= t) lo = mid;
        else hi = mid;
      }
      s += hi;
    } else {  // more than `tile` sequences, empty ones, lie within the tile
      s = sequence_of(a.cu, a.num_seqs, a.tokens, t);
    }
    const int end = min(__ldg(a.cu + s + 1), a.tokens);
    const int64_t pos = (int64_t)__ldg(a.kv_lens + s) - __ldg(a.cu + s + 1) + t;
    run.slot = (int)(pos & (kPage - 1));
    if (t == __ldg(a.cu + s) || run.slot == 0) {
      run.count = min(kPage - run.slot, end - t);
      run.page = page_of(a.table, a.table_stride, a.table_cols, a.num_pages, s, pos, a.status);
    }
  }
  if (i < tile) {
    const uint32_t b = __ballot_sync(0xffffffffu, run.count > 0);
    if ((i & 31) == 0) starts[i >> 5] = b;
  }
  __syncthreads();
  int count = 0, before = 0;
  for (int w = 0; w < tile / 32; ++w) {
    if (w == i / 32) before = count + __popc(starts[w] & ((1u << (i & 31)) - 1));
    count += __popc(starts[w]);
  }
  if (run.count > 0) runs[before] = run;
  __syncthreads();
  return count;
}

// A run's keys (or values) of one head.  Lane 16 z + 2 r + u takes dims 16 u ..
// + 15 of token r of an octet: for every group (G = 2, 4), or of two octets
// (G = 1).  A step takes 2 octets (4).
template <typename T, int G, Order ORDER>
CTI_DEVICE void append_run(const T* __restrict__ rows, int stride, const Run& run,
                           uint8_t* __restrict__ block, int lane) {
  constexpr int kOctets = G == 1 ? 4 : 2;
  constexpr int N = G == 4 ? 4 : 2;  // words that a lane has in each of two vectors of codes
  const int z = lane >> 4, r = (lane >> 1) & 7, u = lane & 1, last = run.slot + run.count - 1;
  const bool odd = r & 1;
  // The lanes of the layout whose words this one has in the end: keys, 4 r + 2 u
  // and the next; values, those of the pair of tokens r / 2 and the dims 16 u + 8
  // (r % 2) .. + 7.
  const int owner0 = ORDER == kKeys ? 4 * r + 2 * u : (4 * u + 2 * (r & 1)) * 4 + (r >> 1);
  constexpr int kNext = ORDER == kKeys ? 16 : 64;  // bytes to the second
  uint8_t* codes = block + (ORDER == kKeys ? 0 : v_codes_at(G));
  for (int nt0 = (run.slot >> 3) / kOctets * kOctets; 8 * nt0 <= last; nt0 += kOctets) {
    const int nt = nt0 + z;  // this lane's octet; G = 1: and the one after the next
    const int src = (8 * nt + r - run.slot) * stride + 16 * u;
    uint4 raw[N][2];
    bool live[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int tau = 8 * (G == 1 ? nt + 2 * j : nt) + r;
      live[j] = tau >= run.slot && tau <= last;
      raw[j][0] = raw[j][1] = make_uint4(0, 0, 0, 0);
      if (live[j]) {
        const uint4* p = reinterpret_cast<const uint4*>(
            rows + src + (G == 1 ? 16 * j * stride : 32 * j));
        raw[j][0] = __ldg(p);
        raw[j][1] = __ldg(p + 1);
      }
    }
    uint32_t w[N][2];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int tau = 8 * (G == 1 ? nt + 2 * j : nt) + r, g = G == 1 ? 0 : j;
      if (G == 1 && !__any_sync(0xffffffffu, live[j])) continue;
      uint32_t s, b;
      quantise<T, ORDER>(raw[j], w[j], s, b);
      if (ORDER == kKeys) {
        if (live[j] && u == 0)
          *reinterpret_cast<uint32_t*>(block + k_meta_at(G) + k_meta_word_at(tau, g, G)) =
              s | b << 16;
      } else {
        // Two tokens share a word: each lane of the pair gets half of the dims.
        const bool pair = live[j] && (tau ^ 1) >= run.slot && (tau ^ 1) <= last;
        const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? w[j][0] : w[j][1], 2);
        const uint32_t mine = s | b << 16, meta = __shfl_xor_sync(0xffffffffu, mine, 2);
        uint8_t* vm = block + v_meta_at(G) + v_meta_half_at(tau, g, G);
        if (live[j] && !pair) {  // an end of the run: its own halves alone
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint16_t*>(codes + v_half_at(tau, g, 4 * u + c, G)) =
                (uint16_t)(w[j][c >> 1] >> (16 * (c & 1)));
          if (u == 0) {
            *reinterpret_cast<uint16_t*>(vm) = (uint16_t)s;
            *reinterpret_cast<uint16_t*>(vm + 4) = (uint16_t)b;
          }
        } else if (pair && u == 0 && !odd) {
          *reinterpret_cast<uint2*>(vm) =
              make_uint2(__byte_perm(mine, meta, 0x5410), __byte_perm(mine, meta, 0x7632));
        }
        const uint32_t even_w = odd ? got : w[j][0], odd_w = odd ? w[j][1] : got;
        w[j][0] = __byte_perm(even_w, odd_w, 0x5410);
        w[j][1] = __byte_perm(even_w, odd_w, 0x7632);
        live[j] = pair;
      }
    }
    const int word0 = nt * G;  // of the lane's words in the layout
    uint8_t* dst = codes + ((word0 >> 2) * 32 + owner0) * 16 + (word0 & 3) * 4;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if constexpr (N == 4) {
        if (live[0])
          *reinterpret_cast<uint4*>(dst + x * kNext) =
              make_uint4(w[0][x], w[1][x], w[2][x], w[3][x]);
      } else if constexpr (G == 2) {
        if (live[0]) *reinterpret_cast<uint2*>(dst + x * kNext) = make_uint2(w[0][x], w[1][x]);
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (live[j]) *reinterpret_cast<uint32_t*>(dst + x * kNext + 8 * j) = w[j][x];
      }
    }
  }
}

// The heads [first, end) of this block: gridDim.y blocks share a tile.
CTI_DEVICE void head_range(const Args& a, int& first, int& end) {
  const int per = (a.kv_heads + gridDim.y - 1) / gridDim.y;
  first = min(a.kv_heads, per * (int)blockIdx.y);
  end = min(a.kv_heads, first + per);
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads, 4)
    kv4_append_runs_kernel(const T* __restrict__ k, const T* __restrict__ v, Args a,
                           uint8_t* __restrict__ pages) {
  __shared__ Run runs[kRunTokens];
  const int lane = lane_id();
  int h0, h1;
  head_range(a, h0, h1);
  const int heads = h1 - h0, units = find_runs(a, blockIdx.x * a.tile, runs) * heads * 2;
  for (int u = warp_id(); u < units; u += kThreads / 32) {
    const int i = (u >> 1) / heads, head = h0 + (u >> 1) - i * heads;
    const Run run = runs[i];
    if (run.page < 0) continue;
    uint8_t* block = pages + (run.page * a.kv_heads + head) * (int64_t)block_bytes(G);
    if ((u & 1) == 0)
      append_run<T, G, kKeys>(k + run.start * a.k_stride + head * (32 * G), (int)a.k_stride, run,
                              block, lane);
    else
      append_run<T, G, kValues>(v + run.start * a.v_stride + head * (32 * G), (int)a.v_stride, run,
                                block, lane);
  }
}

template <typename T, int G>
CTI_DEVICE void read_keys(const uint8_t* __restrict__ block, const Run& run, T* __restrict__ rows,
                          int stride, int lane) {
  constexpr int kOctets = 4 / G;
  const int r = lane >> 2, t = lane & 3, last = run.slot + run.count - 1;
  const int v0 = (run.slot >> 3) / kOctets;
  int tau0 = v0 * kOctets * 8 + r;
  int dst = (tau0 - run.slot) * stride + 8 * t;
  const uint8_t* src = block + (v0 * 32 + lane) * 16;
  const uint32_t* ms = reinterpret_cast<const uint32_t*>(block + k_meta_at(G)) + tau0 * G;
  // Two vectors at a time, all loads first.
  for (; tau0 - r <= last; tau0 += 16 * kOctets, dst += 16 * kOctets * stride, src += 1024, ms += 64) {
    uint4 w4[2];
    uint32_t meta[8];
    bool live[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      w4[u] = make_uint4(0, 0, 0, 0);
      if (tau0 - r + 8 * kOctets * u <= last) w4[u] = __ldg(reinterpret_cast<const uint4*>(src + 512 * u));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int nt = j / G, g = j % G, tau = tau0 + 8 * nt;
      live[j] = tau >= run.slot && tau <= last;
      if (live[j]) meta[j] = __ldg(ms + 8 * nt * G + g);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int nt = j / G, g = j % G;
      const uint32_t w = j % 4 == 0 ? w4[j / 4].x : j % 4 == 1 ? w4[j / 4].y
                         : j % 4 == 2 ? w4[j / 4].z : w4[j / 4].w;
      if (live[j])
        *reinterpret_cast<uint4*>(rows + (dst + 8 * nt * stride) + 32 * g) =
            k_values<T>(w, meta[j]);
    }
  }
}

template <typename T, int G>
CTI_DEVICE void read_values(const uint8_t* __restrict__ block, const Run& run,
                            T* __restrict__ rows, int stride, int lane) {
  constexpr int kOctets = 4 / G;
  const int c = lane >> 2, t = lane & 3, last = run.slot + run.count - 1;
  const int v0 = (run.slot >> 3) / kOctets;
  int tau0 = v0 * kOctets * 8 + 2 * t;  // and the token after it
  int dst = (tau0 - run.slot) * stride + 4 * c;
  const uint8_t* src = block + v_codes_at(G) + (v0 * 32 + lane) * 16;
  const uint2* ms = reinterpret_cast<const uint2*>(block + v_meta_at(G)) + (tau0 >> 1) * G;
  for (; tau0 - 2 * t <= last; tau0 += 16 * kOctets, dst += 16 * kOctets * stride, src += 1024, ms += 32) {
    uint4 w4[2];
    uint2 meta[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      w4[u] = make_uint4(0, 0, 0, 0);
      if (tau0 - 2 * t + 8 * kOctets * u <= last) {
        w4[u] = __ldg(reinterpret_cast<const uint4*>(src + 512 * u));
#pragma unroll
        for (int j = 4 * u; j < 4 * u + 4; ++j) meta[j] = __ldg(ms + 4 * (j / G) * G + j % G);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int nt = j / G, g = j % G, tau = tau0 + 8 * nt;
      const uint32_t w = j % 4 == 0 ? w4[j / 4].x : j % 4 == 1 ? w4[j / 4].y
                         : j % 4 == 2 ? w4[j / 4].z : w4[j / 4].w;
      T* to = rows + (dst + 8 * nt * stride) + 32 * g;
      uint2 even, odd;
      v_values<T>(w, meta[j].x, meta[j].y, even, odd);
      if (tau >= run.slot && tau <= last) *reinterpret_cast<uint2*>(to) = even;
      if (tau + 1 >= run.slot && tau + 1 <= last) *reinterpret_cast<uint2*>(to + stride) = odd;
    }
  }
}

template <typename T, int G>
__global__ void __launch_bounds__(kThreads, 4)
    kv4_read_runs_kernel(const uint8_t* __restrict__ pages, Args a, T* __restrict__ k,
                         T* __restrict__ v) {
  __shared__ Run runs[kRunTokens];
  const int lane = lane_id();
  grid_dependency_wait();
  int h0, h1;
  head_range(a, h0, h1);
  const int heads = h1 - h0, units = find_runs(a, blockIdx.x * a.tile, runs) * heads * 2;
  for (int u = warp_id(); u < units; u += kThreads / 32) {
    const int i = (u >> 1) / heads, head = h0 + (u >> 1) - i * heads;
    const Run run = runs[i];
    const int64_t stride = (u & 1) == 0 ? a.k_stride : a.v_stride;
    T* rows = ((u & 1) == 0 ? k : v) + run.start * stride + head * (32 * G);
    if (run.page < 0) {  // every token of it is outside: zeros
      for (int j = lane; j < run.count * 4 * G; j += 32)
        *reinterpret_cast<uint4*>(rows + (j / (4 * G)) * stride + (j % (4 * G)) * 8) =
            make_uint4(0, 0, 0, 0);
      continue;
    }
    const uint8_t* block = pages + (run.page * a.kv_heads + head) * (int64_t)block_bytes(G);
    if ((u & 1) == 0)
      read_keys<T, G>(block, run, rows, (int)stride, lane);
    else
      read_values<T, G>(block, run, rows, (int)stride, lane);
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
  // A page's tokens are within 2^31 elements of each other.
  if (a.k_stride > kMaxStride || a.v_stride > kMaxStride) return CTI_ERR_UNSUPPORTED;
  if (a.table_stride < a.table_cols) return CTI_ERR_INVALID_ARG;
  return CTI_OK;
}

// The way, the tile and the grid of a call.
struct Launch {
  bool runs;
  dim3 grid;
};
Launch plan(Args& a, int G) {
  Launch l;
  l.runs = a.tokens >= (int64_t)kRunsFrom * a.num_seqs;
  // Longer tiles share the way to their runs among more of them, as long as
  // there are four blocks for each SM.
  a.tile = !l.runs ? kTokens : a.tokens >= kSMs * 4 * kRunTokens ? kRunTokens : kRunTokens / 2;
  const int64_t tiles = ((int64_t)a.tokens + a.tile - 1) / a.tile;
  l.grid = dim3((unsigned)tiles);
  if (l.runs) {
    // Blocks that share a tile by heads: at least four for each SM in all, as
    // long as a block's warps have a run each (two runs start in a tile at
    // the least, with keys and values apart).
    int64_t share = (kSMs * 4 + tiles - 1) / tiles;
    const int64_t most = a.kv_heads * G > 2 ? (a.kv_heads + 1) / 2 : 1;
    l.grid.y = (unsigned)(share > most ? most : share);
  }
  return l;
}

template <typename T, int G>
int launch_append(const void* k, const void* v, Args a, void* pages, cudaStream_t s) {
  const Launch l = plan(a, G);
  auto* kernel = l.runs ? kv4_append_runs_kernel<T, G> : kv4_append_tokens_kernel<T, G>;
  kernel<<<l.grid, kThreads, 0, s>>>(static_cast<const T*>(k), static_cast<const T*>(v), a,
                                     static_cast<uint8_t*>(pages));
  return cudaGetLastError() == cudaSuccess ? CTI_OK : CTI_ERR_CUDA;
}

template <typename T, int G>
int launch_read(const void* pages, Args a, void* k, void* v, cudaStream_t s) {
  const Launch l = plan(a, G);
  auto* kernel = l.runs ? kv4_read_runs_kernel<T, G> : kv4_read_tokens_kernel<T, G>;
  return launch_dependent(kernel, l.grid, dim3(kThreads), 0, s,
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
