// Attention of many new tokens over the 4-bit key/value cache: row tiles of
// 128 on the tensor cores (the definition is in kv4_attention.cu, the format in
// kv4.cuh).
//
// A block takes one or two 128-row tiles (the query heads of one KV head, token
// by token) of a sequence and walks over its pages:
//   warps 0..3 (and 4..7)  softmax of a tile, thread = row.  They lay the
//          tile's queries out in shared memory first: fp16, each row scaled by
//          a power of two.  Per page: the row's 64 scores from TMEM, masked;
//          p = 2^(x - m + 7), m raised (O and l rescaled) only when a score
//          exceeds it by 2^8; P in 16 bits back over the scores.  (The 7 takes p to
//          fp16's range: weights of 2^-21 of the largest keep 11 bits, those
//          below 2^-32 are 0.)
//   4 or 8 warps  unpacking: half of them take a page's keys, half its values,
//          from a ring of page blocks that bulk copies fill, to 16 bits in the
//          swizzled layout of the matrix operands.  Two tiles share the work.
//   1 warp issues S = Q K^T (M 128, N 64), 1 warp O += P V with P from TMEM and
//          V as an MN-major operand.
// All operands are fp16, whatever T.  In bf16 keys, values and P are rounded to 11
// bits, so that the output's own rounding is nearly all of the error.  In fp16, where
// each of these would count as much as the output's, keys and values are two numbers
// each, (16 + n) s' + b and (16 + n) s'' with s' the upper 7 bits of s: both
// exact, but for groups of one sign, whose first number is rounded.  That leaves
// P's rounding and the output's: an error of 0.00029 instead of 0.00048 (keys with
// channels of their own size), for twice the matrix instructions and a half more
// unpacking (5,600 tokens of 16 heads over 5,700 keys: head_dim 32 298 us, 268
// with one number; 64: 345 and 331; 128: 600 and 436).  Keys and
// values are scaled by powers of two first, so that a number keeps its 11 bits
// down to 2^-25 of its page's largest (values: 2^-17).  A page's keys have a
// scaling of their own, which its scores take back.  The values' is the one that O
// is held in, from page to page: it is chosen with the first page (bound of the
// magnitudes at 2^12) and again where a page's bound leaves 2^6 .. 2^15; then O is
// multiplied by the difference, which rounds nothing (fp32 holds O while the
// pages of a sequence's head lie within 2^64 of each other).  So P and the sum l
// know nothing of it.  Every wait is a bounded mbarrier wait; one that runs out
// records its site in the status word and the roles unwind.
//
// Bound by the unpacking for head_dim 128 (without it 554 us become 400 for
// 5,500 tokens of 16 heads over 5,700 keys each), and by the chain S, softmax,
// P V of a page for 32 and 64: about 1.3 us a page.
#include <cfloat>
#include <climits>

#include "kv4_attention.cuh"

namespace cti {
namespace {

using namespace kv4;

constexpr int kTile = 128;

template <typename T, int G, int TILES>
struct Shape {
  // Keys and values as two numbers each.
  static constexpr bool kTwo = Type16<T>::kShift != 3;
  static constexpr int D = 32 * G;
  static constexpr int kRow = D >= 64 ? 128 : 64;  // bytes of an operand row: one swizzle span
  static constexpr int kPanels = D > 64 ? 2 : 1;   // that a row of D takes
  static constexpr int kQPanel = kTile * kRow;
  static constexpr int kQBytes = kPanels * kQPanel;
  static constexpr int kKVPanel = kPage * kRow;
  static constexpr int kKBytes = kPanels * kKVPanel;
  static constexpr int kVAt = (kTwo ? 2 : 1) * kKBytes;  // of a stage: keys, then values
  static constexpr int kStageBytes = 2 * kVAt;
  // Of an SM.  (One tile of two numbers and 64 dims, 96 sequences of 100 rows over 2,000
  // keys: 126 us, two blocks with fewer stages 128; 2 sequences: 22 and 26.)
  static constexpr int kBlocks = TILES == 2 || (kTwo && G >= 2) ? 1 : 2;
  static constexpr int kStages =
      G == 4 ? (kTwo || TILES == 1 ? 2 : 3) : G == 2 ? 3 : 4;
  static constexpr int kRaw = G == 4 && kBlocks == 2 ? 1 : 3;  // page blocks in flight
  static constexpr int kSoftmaxWarps = 4 * TILES;
  static constexpr int kUnpackWarps = kBlocks == 1 ? 8 : 4;
  static constexpr int kThreads = (kSoftmaxWarps + kUnpackWarps + 2) * 32;
  static constexpr uint32_t kTmemCols = TILES == 2 ? 512 : 256;
  // Of a tile: two S / P buffers of 64 columns, then O.
  static constexpr uint32_t kTileCols = 128 + D;
  static_assert(TILES * kTileCols <= kTmemCols, "TMEM budget");
  static constexpr int kInfoBytes = kStages * 48;
  static constexpr int kMetaBytes = 512 * G;  // scales and bases as fp16, by unpacking warp
  static constexpr int kBarBytes = 320;
  static constexpr size_t kSmem =
      1024 + (size_t)TILES * kQBytes + (size_t)kStages * kStageBytes +
      (size_t)kRaw * block_bytes(G) + kInfoBytes + kMetaBytes + kBarBytes;
  static_assert(kSmem <= (kBlocks == 1 ? 232448 : 115000), "shared memory");
};

// What the unpacking warps tell the softmax about a page.
struct alignas(16) PageInfo {
  float scale;        // of its scores: 2^(keys' exponent)
  int keys;           // 64, or 0: not a page
  int v_exponent;     // its values are held as v 2^-v_exponent
  uint64_t nan_v[4];  // bit per key: a value that is not finite (pages that some rows see in part)
};

// What the swizzle of operand rows of ROW bytes flips in a byte's place in row r.
template <int ROW>
CTI_DEVICE int swizzle_of(int r) {
  return ROW == 128 ? (r & 7) << 4 : (r >> 1 & 3) << 4;
}

// Matrix descriptor of an operand tile, 8-row atoms stacked along its rows: K-major
// for Q and K, MN-major (each row a key) for V.  The stride field holds an
// atom's bytes; the leading one the bytes between the panels of a wide V.
template <int ROW>
CTI_DEVICE uint64_t tile_desc(uint32_t saddr, uint32_t panel = 8 * ROW) {
  constexpr uint64_t atom = 8 * ROW;
  return (uint64_t)((saddr >> 4) & 0x3fffu) | (uint64_t)(panel >> 4) << 16 | (atom >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)(ROW == 128 ? 2 : 4) << 61;
}

// The larger of both halves of two numbers of T that are not negative; a NaN
// counts nothing.
template <typename T>
CTI_DEVICE uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (Type16<T>::kShift == 3)
    asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else
    asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A scale of fp16 as two: its upper 7 bits, and the other 4.  A sum (16 + n) top + b
// of a group whose values are not of one sign is a multiple of s 2^-7 or more and
// below 16 s, so 11 bits hold it; (16 + n) rest has 9.
struct TwoScales {
  uint32_t top, rest;
  CTI_DEVICE explicit TwoScales(uint32_t s) : top(s & 0xfff0fff0u) {
    const __half2 d = __hsub2_rn(*reinterpret_cast<__half2*>(&s), *reinterpret_cast<__half2*>(&top));
    rest = *reinterpret_cast<const uint32_t*>(&d);
  }
};

// a b of both halves in fp16.
CTI_DEVICE uint32_t mul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2_rn(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 16 TMEM columns and their wait in one statement, as the 32-column form.
CTI_DEVICE void tmem_ld_x16_sync(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

template <typename T, int G, int TILES>
__global__ void __launch_bounds__(Shape<T, G, TILES>::kThreads, Shape<T, G, TILES>::kBlocks)
    kv4_tiles_kernel(const T* __restrict__ q, const uint8_t* __restrict__ pages, const Args a,
                     T* __restrict__ out) {
  using Y = Type16<T>;
  using Z = Shape<T, G, TILES>;
  constexpr int D = Z::D;
  constexpr int S = Z::kStages, R = Z::kRaw;
  constexpr int kRow = Z::kRow;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + TILES * Z::kQBytes;  // [S] x {K, V}
  uint8_t* sRaw = sKV + (size_t)S * Z::kStageBytes;  // [R] page blocks
  PageInfo* info = reinterpret_cast<PageInfo*>(sRaw + (size_t)R * block_bytes(G));
  uint32_t* sMeta = reinterpret_cast<uint32_t*>(info + S);
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(sMeta + Z::kMetaBytes / 4);  // [S]
  uint64_t* kv_empty = kv_full + S;                           // [S] PV of every tile done
  uint64_t* q_full = kv_empty + S;                            // [TILES] (4 softmax warps)
  uint64_t* q_empty = q_full + TILES;                         // [TILES] last S done
  uint64_t* o_empty = q_empty + TILES;                        // [TILES] O read (4 warps)
  uint64_t* s_full = o_empty + TILES;                         // [TILES][2]
  uint64_t* p_full = s_full + 2 * TILES;                      // [TILES][2] (4 warps)
  uint64_t* pv_done = p_full + 2 * TILES;                     // [TILES][2]
  uint64_t* raw_full = pv_done + 2 * TILES;                   // [R]
  uint64_t* raw_empty = raw_full + R;                         // [R] (unpacking warps)
  uint64_t* drain = raw_empty + R;                            // [2] each issuer's last
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * S + 9 * TILES + 2 * R + 2) * 8 + 8 <= Z::kBarBytes, "barrier area");

  const int warp = warp_id(), lane = lane_id();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&kv_full[i], Z::kUnpackWarps);
      mbar_init(&kv_empty[i], TILES);
    }
    for (int i = 0; i < TILES; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&q_empty[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < 2 * TILES; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < R; ++i) {
      mbar_init(&raw_full[i], 1);
      mbar_init(&raw_empty[i], Z::kUnpackWarps);
    }
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  // Everything read below may come from the kernel before; tensor memory too may
  // still be that kernel's, which must not wait for ours.
  grid_dependency_wait();
  if (warp == Z::kSoftmaxWarps + Z::kUnpackWarps) {
    tmem_alloc(tmem_slot, Z::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // ---- the sequence ----
  const int s = (int)a.by_kv_heads(blockIdx.x), kvh = (int)blockIdx.x - s * a.kv_heads;
  const int group = a.group;
  const int begin = __ldg(a.cu + s), end = __ldg(a.cu + s + 1);
  const int len = max(__ldg(a.kv_lens + s), 0);
  const bool sound = begin >= 0 && end <= a.tokens && end >= begin;
  if (!sound && threadIdx.x == 0) raise_status(a.status, CTI_ERR_INVALID_ARG, s);
  const int n_new = sound ? end - begin : 0;
  const int first = len - n_new;
  const int rows = n_new * group;
  int limit = len;
  if (limit > a.table_cols * kPage || (limit > 0 && a.num_pages <= 0)) {
    if (threadIdx.x == 0 && rows > 0) raise_status(a.status, CTI_ERR_BOUNDS, s);
    limit = a.num_pages <= 0 ? 0 : a.table_cols * kPage;
  }
  constexpr int kRows = TILES * kTile;
  const int ntiles = (rows + kRows - 1) / kRows;

  // The pages [p0, p0 + np) of this block for the rows from row0 on, the keys
  // that some row and that every row sees.
  struct Range {
    int p0, np, most, all;
  };
  auto range_of = [&](int tile) {
    const int row0 = tile * kRows, row_last = min(rows, row0 + kRows) - 1;
    Range r;
    r.most = max(a.causal ? min(first + (int)a.by_group(row_last) + 1, limit) : limit, 0);
    r.all = a.causal ? min(first + (int)a.by_group(row0) + 1, limit) : limit;
    r.p0 = 0;
    r.np = (r.most + kPage - 1) / kPage;
    if (gridDim.z > 1) {  // the last block takes what the caller's bound left out
      r.p0 = min(r.np, (int)blockIdx.z * a.chunk);
      r.np = (blockIdx.z == gridDim.z - 1 ? r.np : min(r.np, r.p0 + a.chunk)) - r.p0;
    }
    return r;
  };

  if (warp < Z::kSoftmaxWarps) {
    // ---------------- softmax ----------------
    const int i = warp >> 2, wq = warp & 3;
    const int r = wq * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(wq * 32) << 16) + i * Z::kTileCols;
    uint8_t* myq = sQ + i * Z::kQBytes;
    const int swizzle = swizzle_of<kRow>(r);
    int it = 0, g = 0;
    bool ok = true;
    for (int tile = blockIdx.y; ok && tile < ntiles; tile += gridDim.y, ++it) {
      const Range rg = range_of(tile);
      if (i > 0 && tile * kRows + i * kTile >= rows) break;
      const int row = tile * kRows + i * kTile + r;
      const bool live = row < rows;
      const int tok = live ? (int)a.by_group(row) : 0;
      const int head = kvh * group + (live ? row - tok * group : 0);
      const int64_t at = (int64_t)(begin + tok) * a.heads + head;
      // A row of no query sees everything: nothing is masked for it.
      const int sees = !live ? INT_MAX : a.causal ? min(first + tok + 1, limit) : limit;
      // Queries: the row's largest magnitude, then fp16 in [2^14, 2^15) at most.
      const uint4* src =
          reinterpret_cast<const uint4*>(q + (begin + tok) * a.q_stride + (int64_t)head * D);
      float most_q = 0.0f;
      if (live) {
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint4 v = __ldg(src + c);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            most_q = max3f(most_q, fabsf(Y::low(w[j])), fabsf(Y::high(w[j])));
        }
      }
      const int k = query_exponent(most_q, a);
      const float up = power_of_two(k) * a.sign;
      const float down = a.scale_m * power_of_two(min(a.scale_e - k, 128));
      if (!__all_sync(0xffffffffu,
                      mbar_wait(&q_empty[i], (uint32_t)(it & 1) ^ 1u, a.status, 0x710, abort_flag)))
        break;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live) v = __ldg(src + c);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          h[j] = Type16<__half>::pack(Y::low(w[j]) * up, Y::high(w[j]) * up);
        const int panel = c * 16 / kRow, off = c * 16 % kRow;
        *reinterpret_cast<uint4*>(myq + panel * Z::kQPanel + r * kRow + (off ^ swizzle)) =
            make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[i]);

      float m = -INFINITY, l = 0.0f;  // m in powers of 2
      int unit = 0;                   // O is held in units of 2^unit
      for (int j = 0; j < rg.np; ++j, ++g) {
        const int b = g & 1, st = g % S;
        // kv_full has completed once s_full has; waited for here to see the info.
        if (!__all_sync(0xffffffffu,
                        mbar_wait(&kv_full[st], (uint32_t)((g / S) & 1), a.status, 0x711,
                                  abort_flag) &&
                            mbar_wait(&s_full[2 * i + b], (uint32_t)((g >> 1) & 1), a.status,
                                      0x712, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sb = lanes + 64u * b;
        const PageInfo pi = info[st];
        const int key0 = (rg.p0 + j) * kPage;
        const uint64_t nan_v = pi.nan_v[0] | pi.nan_v[1] | pi.nan_v[2] | pi.nan_v[3];
        const int lim = min(sees - key0, pi.keys);
        if (nan_v != 0 || !__all_sync(0xffffffffu, lim >= kPage)) {
          // Scores that do not count, put back before the pass below (a short loop
          // on its own keeps that pass's instructions few).
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t x[16];
            tmem_ld_x16_sync(sb + 16 * c, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              if (nan_v >> (16 * c + e) & 1) x[e] = 0x7fffffffu;
              if (16 * c + e >= lim) x[e] = __float_as_uint(-INFINITY);
            }
            tmem_st_32x32b_x16(sb + 16 * c, x);
          }
          tmem_st_wait();
        }
        // The scores go through registers 32 at a time, twice: short loops, whose
        // instructions stay at hand while warps of other roles run between
        // (unrolled, with one reading of all 64: 545 us instead of 502 for
        // 5,500 tokens of 16 heads of 128 over 5,700 keys each).
        float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t x[32];
          tmem_ld_32x32b_x32_sync(sb + 32 * c, x);
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            mx = max3f(mx, __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
            mx1 = max3f(mx1, __uint_as_float(x[e + 2]), __uint_as_float(x[e + 3]));
          }
        }
        const float factor = fmaxf(down * pi.scale, 1e-37f);  // -inf stays -inf, and 2^37 next to 0
        mx = fmaxf(mx, mx1) * factor;
        float corr = 1.0f;
        if (mx - m > kSlack) {
          corr = ex2_approx(m - mx);
          m = mx;
        }
        const int rise = j > 0 ? pi.v_exponent - unit : 0;  // the same for the block
        unit = pi.v_exponent;
        if (rise != 0 || __any_sync(0xffffffffu, corr != 1.0f)) {
          l *= corr;
          if (j > 0) {
            const float corr_o = corr * power_of_two(-max(-127, min(rise, 126)));
            // O holds the tile's pages up to g - 1: wait for their PV.
            if (!__all_sync(0xffffffffu,
                            mbar_wait(&pv_done[2 * i + (b ^ 1)], (uint32_t)(((g - 1) >> 1) & 1),
                                      a.status, 0x713, abort_flag))) {
              ok = false;
              break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 2 * G; ++c) {
              uint32_t o[16];
              tmem_ld_x16_sync(lanes + 128 + 16 * c, o);
#pragma unroll
              for (int d = 0; d < 16; ++d) o[d] = __float_as_uint(__uint_as_float(o[d]) * corr_o);
              tmem_st_32x32b_x16(lanes + 128 + 16 * c, o);
            }
          }
        }
        const float noff = m == -INFINITY ? 0.0f : kPUnitFp16 - m;
        const uint64_t factor2 = f2_pack(factor, factor), noff2 = f2_pack(noff, noff);
        uint64_t sum_a = f2_pack(0.0f, 0.0f), sum_b = sum_a;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t x[32];
          tmem_ld_32x32b_x32_sync(sb + 32 * c, x);
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(x[2 * e]),
                                     __uint_as_float(x[2 * e + 1])),
                             factor2, noff2),
                      x0, x1);
            const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            if (e & 1) sum_b = f2_add(sum_b, f2_pack(p0, p1));
            else sum_a = f2_add(sum_a, f2_pack(p0, p1));
            pk[e] = Type16<__half>::pack(p0, p1);
          }
          tmem_st_32x32b_x16(sb + 16 * c, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * i + b]);
        float s0, s1;
        f2_unpack(f2_add(sum_a, sum_b), s0, s1);
        l += s0 + s1;
      }
      if (!ok) break;
      // ---- the rows ----
      if (rg.np > 0) {
        if (!__all_sync(0xffffffffu,
                        mbar_wait(&pv_done[2 * i + ((g - 1) & 1)], (uint32_t)(((g - 1) >> 1) & 1),
                                  a.status, 0x714, abort_flag)))
          break;
        tc_fence_after();
      }
      // Two factors: their product may leave fp32's range.
      const float inv = l == 0.0f ? 0.0f : 1.0f / l, up_o = power_of_two(unit);
      const int64_t ws = (int64_t)blockIdx.z * a.tokens * a.heads + at;
#pragma unroll 1
      for (int c = 0; c < 2 * G; ++c) {
        uint32_t o[16];
        if (rg.np > 0) {
          tmem_ld_x16_sync(lanes + 128 + 16 * c, o);
        } else {
#pragma unroll
          for (int d = 0; d < 16; ++d) o[d] = 0;
        }
        if (!live) continue;
#pragma unroll
        for (int d = 0; d < 16; ++d)
          o[d] = __float_as_uint(__uint_as_float(o[d]) * inv * up_o);
        if (gridDim.z == 1) {
          uint4* dst = reinterpret_cast<uint4*>(out + at * D + 16 * c);
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              w[x] = Y::pack(__uint_as_float(o[8 * d + 2 * x]),
                             __uint_as_float(o[8 * d + 2 * x + 1]));
            dst[d] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else if (rg.np > 0) {
          uint4* dst = reinterpret_cast<uint4*>(a.ws_o + ws * D + 16 * c);
#pragma unroll
          for (int d = 0; d < 4; ++d)
            dst[d] = make_uint4(o[4 * d], o[4 * d + 1], o[4 * d + 2], o[4 * d + 3]);
        }
      }
      if (live && gridDim.z > 1) a.ws_ml[ws] = make_float2(m, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[i]);
    }
  } else if (warp < Z::kSoftmaxWarps + Z::kUnpackWarps) {
    // ---------------- unpacking ----------------
    constexpr int kEach = Z::kUnpackWarps / 2;  // warps for keys, and for values
    constexpr int kVecs = 2 * G / kEach;        // vectors of codes that each takes
    const int dw = warp - Z::kSoftmaxWarps;
    const bool keys = dw < kEach;
    const int part = keys ? dw : dw - kEach;
    const int hi = lane >> 2, lo = lane & 3;
    const int32_t* table = a.table + s * a.table_stride;
    const uint8_t* base = pages + (int64_t)kvh * block_bytes(G);
    const int64_t page_stride = (int64_t)a.kv_heads * block_bytes(G);
    // Bytes of this lane's pieces in an octet of rows, for an even group; an odd
    // one differs in bit 6.  Keys: row hi, dims 8 lo .. + 7.  Values: rows
    // 2 lo and 2 lo + 1, dims 4 hi .. + 3.
    const int at_k = hi * kRow + (16 * lo ^ swizzle_of<kRow>(hi));
    const int at_v0 = 2 * lo * kRow + (8 * hi ^ swizzle_of<kRow>(2 * lo));
    const int at_v1 = (2 * lo + 1) * kRow + (8 * hi ^ swizzle_of<kRow>(2 * lo + 1));
    int g = 0, asked = 0;  // pages unpacked, and (the first of these warps) copies asked for
    bool ok = true;
    for (int tile = blockIdx.y; ok && tile < ntiles; tile += gridDim.y) {
      const Range rg = range_of(tile);
      int ids = 0;
      // The values' exponent, and the largest it was (INT_MIN: no page has set it).
      int unit = 0, unit_most = INT_MIN;
      for (int j = 0; j < rg.np; ++j, ++g) {
        if ((j & 31) == 0) {
          ids = j + lane < rg.np ? __ldg(table + rg.p0 + j + lane) : 0;
          if (ids < 0 || ids >= a.num_pages) {
            raise_status(a.status, CTI_ERR_BOUNDS, s);
            ids = -1;
          }
        }
        // The first warp keeps R pages of these 32 in flight.
        if (dw == 0) {
          const int ahead = min(g + R, g - j + min(rg.np, (j & ~31) + 32));
          for (; asked < ahead; ++asked) {
            const int slot = asked % R, id = __shfl_sync(0xffffffffu, ids, (asked - g + j) & 31);
            ok = __all_sync(0xffffffffu, mbar_wait(&raw_empty[slot],
                                                   (uint32_t)((asked / R) & 1) ^ 1u, a.status,
                                                   0x722, abort_flag));
            if (!ok) break;
            if (lane == 0) {
              mbar_arrive_expect_tx(&raw_full[slot], block_bytes(G));
              bulk_load(sRaw + slot * block_bytes(G), base + max(id, 0) * page_stride,
                        block_bytes(G), &raw_full[slot]);
            }
          }
          if (!ok) break;
        }
        const bool is_page = __shfl_sync(0xffffffffu, ids, j & 31) >= 0;
        const int key0 = (rg.p0 + j) * kPage;
        const int most = is_page ? rg.most - key0 : 0;  // keys of the page that some row sees
        const bool whole = is_page && key0 + kPage <= rg.all;
        const int st = g % S;
        uint8_t* dst = sKV + (size_t)st * Z::kStageBytes;
        const uint8_t* blk = sRaw + (g % R) * block_bytes(G);
        ok = __all_sync(0xffffffffu,
                        mbar_wait(&raw_full[g % R], (uint32_t)((g / R) & 1), a.status, 0x720,
                                  abort_flag) &&
                            mbar_wait(&kv_empty[st], (uint32_t)((g / S) & 1) ^ 1u, a.status,
                                      0x721, abort_flag));
        if (!ok) break;
        // The part's scales and bases: words of (s, b) of a key, or pairs of words
        // (s of two tokens, b of both).  A bound of the page's magnitudes, 31 max
        // s + max |b| (at most 8 times the largest), gives its scaling; all warps
        // of the part find the same, page by page.
        const uint32_t* raw_meta = reinterpret_cast<const uint32_t*>(
            blk + (keys ? k_meta_at(G) : v_meta_at(G)));
        uint32_t most_s = 0, most_b = 0;  // of keys: both in most_s
#pragma unroll
        for (int x = 0; x < (G + 1) / 2; ++x) {
          constexpr int kWords = G == 1 ? 2 : 4;  // side by side, of a lane
          const int i = (32 * x + lane) * kWords;
          uint32_t w[4] = {0, 0, 0, 0};
          if constexpr (G == 1) {
            const uint2 m2 = *reinterpret_cast<const uint2*>(raw_meta + i);
            w[0] = m2.x, w[1] = m2.y;
          } else {
            const uint4 m4 = *reinterpret_cast<const uint4*>(raw_meta + i);
            w[0] = m4.x, w[1] = m4.y, w[2] = m4.z, w[3] = m4.w;
          }
#pragma unroll
          for (int y = 0; y < kWords; ++y) {
            w[y] &= 0x7fff7fffu;
            if (!whole) {
              const int tau = keys ? (i + y) / G : (i + y) / (2 * G) * 2;
              if (tau >= most) w[y] = 0;
              else if (!keys && tau + 1 >= most) w[y] &= 0xffffu;
            }
            if (keys || (y & 1) == 0) most_s = max2<T>(most_s, w[y]);
            else most_b = max2<T>(most_b, w[y]);
          }
        }
        const float top_s = keys ? Y::low(most_s) : fmaxf(Y::low(most_s), Y::high(most_s));
        const float top_b = keys ? Y::high(most_s) : fmaxf(Y::low(most_b), Y::high(most_b));
        const float top = __uint_as_float(__reduce_max_sync(
            0xffffffffu, __float_as_uint(fminf(fmaf(31.0f, top_s, top_b), FLT_MAX))));
        const int top_e = (int)(__float_as_uint(top) >> 23) - 127;
        int e;
        if (keys) {
          e = top > 0.0f ? max(-116, top_e - 14) : 0;  // to 2^14
        } else {
          // O, below 2^30 for each key, stays finite in a unit 2^64 below its largest.
          if (top > 0.0f && (unit_most == INT_MIN || top_e - unit < 6 || top_e - unit >= 15)) {
            unit = max(-116, top_e - 12);
            if (unit_most != INT_MIN) unit = max(unit, unit_most - 64);
            unit_most = max(unit, unit_most);
          }
          e = unit;
        }
        const float down = power_of_two(-e);
        // This warp's own, scaled and as fp16.
        uint32_t* meta = sMeta + (warp - Z::kSoftmaxWarps) * (32 * kVecs);
        uint64_t nan_bits = 0;
#pragma unroll
        for (int x = 0; x < kVecs; ++x) {
          const int i = 32 * (part * kVecs + x) + lane;
          uint32_t w = raw_meta[i];
          if (!keys && !whole) {
            // Behind the last key: zero.  Not finite: zero, and the softmax is told.
            const int tau = 2 * (i / (2 * G));
            constexpr uint32_t inf = Inf16<T>::kBits;
            uint32_t n = ((w & inf) == inf ? 1u : 0u) | ((w >> 16 & inf) == inf ? 2u : 0u);
            n |= __shfl_xor_sync(0xffffffffu, n, 1);  // the other of s and b
            n &= (tau < most ? 1u : 0u) | (tau + 1 < most ? 2u : 0u);
            w &= ((n & 1) || tau >= most ? 0u : 0xffffu) |
                 ((n & 2) || tau + 1 >= most ? 0u : 0xffff0000u);
            nan_bits |= (uint64_t)n << tau;
          }
          meta[32 * x + lane] =
              Type16<__half>::pack(Y::low(w) * down, Y::high(w) * down);
        }
        __syncwarp();
        if (keys) {
          if (part == 0 && lane == 0) {
            info[st].scale = power_of_two(e);
            info[st].keys = is_page ? kPage : 0;
          }
#pragma unroll 1
          for (int x = 0; x < kVecs; ++x) {
            const int v = part * kVecs + x, nt0 = 4 * v / G;
            const uint4 w4 = *reinterpret_cast<const uint4*>(blk + (v * 32 + lane) * 16);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
            const uint32_t* mv = meta + 32 * x + hi * G;
            uint32_t sb[4];
            if constexpr (G == 4) {
              const uint4 m4 = *reinterpret_cast<const uint4*>(mv);
              sb[0] = m4.x, sb[1] = m4.y, sb[2] = m4.z, sb[3] = m4.w;
            } else {
#pragma unroll
              for (int y = 0; y < 4; ++y) sb[y] = mv[8 * (y / G) * G + y % G];
            }
            uint8_t* to = dst + nt0 * 8 * kRow;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int nt = y / G, gr = y % G;  // nt: octets past nt0
              const uint32_t s2 = __byte_perm(sb[y], sb[y], 0x1010);
              const uint32_t b2 = __byte_perm(sb[y], sb[y], 0x3232);
              uint8_t* row = to + (gr >> 1) * Z::kKVPanel + nt * 8 * kRow + (at_k ^ 64 * (gr & 1));
              uint32_t o[4];
              if constexpr (Z::kTwo) {
                const TwoScales two(s2);
                uint32_t rest[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                  const uint32_t c = code_pair<__half>(w[y], p);
                  o[p] = fma2<__half>(c, two.top, b2);
                  rest[p] = mul2(c, two.rest);
                }
                *reinterpret_cast<uint4*>(row + Z::kKBytes) =
                    make_uint4(rest[0], rest[1], rest[2], rest[3]);
              } else {
#pragma unroll
                for (int p = 0; p < 4; ++p)
                  o[p] = fma2<__half>(code_pair<__half>(w[y], p), s2, b2);
              }
              *reinterpret_cast<uint4*>(row) = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
        } else {
          uint8_t* vt = dst + Z::kVAt;
#pragma unroll 1
          for (int x = 0; x < kVecs; ++x) {
            const int v = part * kVecs + x, nt0 = 4 * v / G;
            const uint4 w4 =
                *reinterpret_cast<const uint4*>(blk + v_codes_at(G) + (v * 32 + lane) * 16);
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
            const uint2* mv = reinterpret_cast<const uint2*>(meta + 32 * x) + lo * G;
            uint2 sb[4];
            if constexpr (G == 1) {
#pragma unroll
              for (int y = 0; y < 4; ++y) sb[y] = mv[4 * y];
            } else {
#pragma unroll
              for (int y = 0; y < 4; y += 2) {
                const uint4 m4 =
                    *reinterpret_cast<const uint4*>(mv + 4 * (y / G) * G + y % G);
                sb[y] = make_uint2(m4.x, m4.y);
                sb[y + 1] = make_uint2(m4.z, m4.w);
              }
            }
            uint8_t* to = vt + nt0 * 8 * kRow;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int nt = y / G, gr = y % G;
              uint32_t o[4];
              uint8_t* row = to + (gr >> 1) * Z::kKVPanel + nt * 8 * kRow;
              if constexpr (Z::kTwo) {
                const TwoScales two(sb[y].x);
                uint32_t rest[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                  const uint32_t c = code_pair<__half>(w[y], p);
                  o[p] = fma2<__half>(c, two.top, sb[y].y);
                  rest[p] = mul2(c, two.rest);
                }
                uint8_t* low = row + Z::kKBytes;
                *reinterpret_cast<uint2*>(low + (at_v0 ^ 64 * (gr & 1))) = make_uint2(
                    __byte_perm(rest[0], rest[1], 0x5410), __byte_perm(rest[2], rest[3], 0x5410));
                *reinterpret_cast<uint2*>(low + (at_v1 ^ 64 * (gr & 1))) = make_uint2(
                    __byte_perm(rest[0], rest[1], 0x7632), __byte_perm(rest[2], rest[3], 0x7632));
              } else {
#pragma unroll
                for (int p = 0; p < 4; ++p)
                  o[p] = fma2<__half>(code_pair<__half>(w[y], p), sb[y].x, sb[y].y);
              }
              *reinterpret_cast<uint2*>(row + (at_v0 ^ 64 * (gr & 1))) =
                  make_uint2(__byte_perm(o[0], o[1], 0x5410), __byte_perm(o[2], o[3], 0x5410));
              *reinterpret_cast<uint2*>(row + (at_v1 ^ 64 * (gr & 1))) =
                  make_uint2(__byte_perm(o[0], o[1], 0x7632), __byte_perm(o[2], o[3], 0x7632));
            }
          }
          if (!whole) {
            const uint32_t n0 = __reduce_or_sync(0xffffffffu, (uint32_t)nan_bits);
            const uint32_t n1 = __reduce_or_sync(0xffffffffu, (uint32_t)(nan_bits >> 32));
            nan_bits = (uint64_t)n1 << 32 | n0;
          }
          if (lane == 0) {
            info[st].nan_v[part] = nan_bits;
            if (kEach == 2) info[st].nan_v[part + 2] = 0;
            if (part == 0) info[st].v_exponent = e;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&raw_empty[g % R]);
          mbar_arrive(&kv_full[st]);
        }
      }
    }
    // Let the copies in flight land before the block can end.
    if (dw == 0)
      for (int i = max(0, asked - R); i < asked; ++i)
        mbar_wait(&raw_full[i % R], (uint32_t)((i / R) & 1), a.status, 0x723, nullptr);
  } else if (warp == Z::kSoftmaxWarps + Z::kUnpackWarps) {
    // ---------------- S issuer ----------------
    if (lane == 0) {
      // fp16 operands, fp32 sums; M 128, N 64
      constexpr uint32_t id_s = (1u << 4) | ((kPage >> 3) << 17) | ((kTile >> 4) << 24);
      const uint32_t q_addr = smem_u32(sQ), kv_addr = smem_u32(sKV);
      int it = 0, g = 0;
      bool ok = true, any = false;
      for (int tile = blockIdx.y; ok && tile < ntiles; tile += gridDim.y, ++it) {
        const Range rg = range_of(tile);
        const int tiles = TILES == 2 && rows - tile * kRows <= kTile ? 1 : TILES;
#pragma unroll
        for (int i = 0; i < TILES; ++i)
          ok = ok && (i >= tiles || mbar_wait(&q_full[i], (uint32_t)(it & 1), a.status, 0x730,
                                                 abort_flag));
        for (int j = 0; ok && j < rg.np; ++j, ++g) {
          const int st = g % S, b = g & 1;
          ok = mbar_wait(&kv_full[st], (uint32_t)((g / S) & 1), a.status, 0x731, abort_flag);
#pragma unroll
          for (int i = 0; i < TILES; ++i) {
            if (!ok || i >= tiles) break;
            // The buffer's last reader is the PV of page g - 2.
            ok = mbar_wait(&pv_done[2 * i + b], (uint32_t)((g >> 1) & 1) ^ 1u, a.status, 0x732,
                           abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t qa = q_addr + i * Z::kQBytes, ka = kv_addr + st * Z::kStageBytes;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const int panel = kk * 32 / kRow, off = kk * 32 % kRow;
              umma_bf16(tmem + i * Z::kTileCols + 64u * b,
                        tile_desc<kRow>(qa + panel * Z::kQPanel + off),
                        tile_desc<kRow>(ka + panel * Z::kKVPanel + off), id_s, kk != 0 ? 1u : 0u);
              if (Z::kTwo)
                umma_bf16(tmem + i * Z::kTileCols + 64u * b,
                          tile_desc<kRow>(qa + panel * Z::kQPanel + off),
                          tile_desc<kRow>(ka + Z::kKBytes + panel * Z::kKVPanel + off), id_s, 1u);
            }
            umma_commit(&s_full[2 * i + b]);
            any = true;
          }
        }
        if (!ok) break;
        for (int i = 0; i < TILES; ++i) {
          if (any) umma_commit(&q_empty[i]);
          else mbar_arrive(&q_empty[i]);
        }
      }
      if (any) {
        umma_commit(&drain[0]);
        mbar_wait(&drain[0], 0, a.status, 0x733, nullptr);
      }
    }
  } else {
    // ---------------- PV issuer ----------------
    if (lane == 0) {
      // fp16 operands, fp32 sums; V MN-major
      constexpr uint32_t id_pv = (1u << 4) | (1u << 16) | ((D >> 3) << 17) | ((kTile >> 4) << 24);
      const uint32_t kv_addr = smem_u32(sKV);
      int it = 0, g = 0;
      bool ok = true, any = false;
      for (int tile = blockIdx.y; ok && tile < ntiles; tile += gridDim.y, ++it) {
        const Range rg = range_of(tile);
        const int tiles = TILES == 2 && rows - tile * kRows <= kTile ? 1 : TILES;
        for (int j = 0; ok && j < rg.np; ++j, ++g) {
          const int st = g % S, b = g & 1;
#pragma unroll
          for (int i = 0; i < TILES; ++i) {
            if (!ok || i >= tiles) break;
            if (j == 0)  // the last tile's O has been read
              ok = mbar_wait(&o_empty[i], (uint32_t)(it & 1) ^ 1u, a.status, 0x740, abort_flag);
            ok = ok && mbar_wait(&p_full[2 * i + b], (uint32_t)((g >> 1) & 1), a.status, 0x741,
                                 abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t pbuf = tmem + i * Z::kTileCols + 64u * b;
            const uint32_t ocol = tmem + i * Z::kTileCols + 128u;
            const uint32_t va = kv_addr + st * Z::kStageBytes + Z::kVAt;
#pragma unroll
            for (int kk = 0; kk < kPage / 16; ++kk) {
              constexpr uint32_t panel = Z::kPanels == 2 ? Z::kKVPanel : 8 * kRow;
              umma_bf16_ts(ocol, pbuf + kk * 8, tile_desc<kRow>(va + kk * 16 * kRow, panel), id_pv,
                           j == 0 && kk == 0 ? 0u : 1u);
              if (Z::kTwo)
                umma_bf16_ts(ocol, pbuf + kk * 8,
                             tile_desc<kRow>(va + Z::kKBytes + kk * 16 * kRow, panel), id_pv, 1u);
            }
            umma_commit(&pv_done[2 * i + b]);
            umma_commit(&kv_empty[st]);
            any = true;
          }
          for (int i = tiles; ok && i < TILES; ++i) mbar_arrive(&kv_empty[st]);
        }
        // A tile without pages leaves O alone, but its turn counts.
        for (int i = 0; ok && rg.np == 0 && i < tiles; ++i)
          ok = mbar_wait(&o_empty[i], (uint32_t)(it & 1) ^ 1u, a.status, 0x742, abort_flag);
      }
      if (any) {
        umma_commit(&drain[1]);
        mbar_wait(&drain[1], 0, a.status, 0x743, nullptr);
      }
    }
  }

  __syncthreads();
  if (warp == Z::kSoftmaxWarps + Z::kUnpackWarps) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, Z::kTmemCols);
  }
  if (gridDim.z > 1 && blockIdx.z == 0 && blockIdx.y == 0) {
    // Here, not where the offsets are first read, so that the roles' registers stay theirs.
    const int seq = (int)a.by_kv_heads(blockIdx.x);
    const int from = __ldg(a.cu + seq), to = __ldg(a.cu + seq + 1);
    if (from < 0 || to > a.tokens || to < from)
      refuse_rows(a.ws_ml, max(from, 0), min(to, a.tokens), a.heads, a.group,
                  (int)blockIdx.x - seq * a.kv_heads);
  }
}

template <typename T, int G, int TILES>
int launch(const void* q, const void* pages, const Args& a, int64_t y, int splits, void* out,
           cudaStream_t s) {
  using Z = Shape<T, G, TILES>;
  static uint64_t configured = 0;
  if (ensure_smem_limit(kv4_tiles_kernel<T, G, TILES>, (int)Z::kSmem, configured) != cudaSuccess)
    return CTI_ERR_CUDA;
  const dim3 grid((unsigned)((int64_t)a.num_seqs * a.kv_heads), (unsigned)(y < 65535 ? y : 65535),
                  (unsigned)splits);
  return launch_dependent(kv4_tiles_kernel<T, G, TILES>, grid, dim3(Z::kThreads), Z::kSmem, s,
                          static_cast<const T*>(q), static_cast<const uint8_t*>(pages), a,
                          static_cast<T*>(out)) == cudaSuccess
             ? CTI_OK
             : CTI_ERR_CUDA;
}

template <typename T, int G>
int launch_shape(const void* q, const void* pages, const Args& a, int tiles, int64_t y, int splits,
                 void* out, cudaStream_t s) {
  if constexpr (G > 1)
    if (tiles == 2) return launch<T, G, 2>(q, pages, a, y, splits, out, s);
  return launch<T, G, 1>(q, pages, a, y, splits, out, s);
}

template <typename T>
int launch_dim(const void* q, const void* pages, const Args& a, int head_dim, int tiles, int64_t y,
               int splits, void* out, cudaStream_t s) {
  return head_dim == 32   ? launch_shape<T, 1>(q, pages, a, tiles, y, splits, out, s)
         : head_dim == 64 ? launch_shape<T, 2>(q, pages, a, tiles, y, splits, out, s)
                          : launch_shape<T, 4>(q, pages, a, tiles, y, splits, out, s);
}

}  // namespace

int kv4::launch_tiles(const void* q, const void* pages, const Args& a, int dtype, int head_dim,
                      int tiles, int64_t y, int splits, void* out, cudaStream_t s) {
  return dtype == CTI_DTYPE_BF16
             ? launch_dim<__nv_bfloat16>(q, pages, a, head_dim, tiles, y, splits, out, s)
             : launch_dim<__half>(q, pages, a, head_dim, tiles, y, splits, out, s);
}

}  // namespace cti
