// Attention of new tokens over the 4-bit key/value cache (format: kv4.cuh):
//   out[t, h, :] = sum_j softmax_j(scale q[t, h, :] . k_j) v_j
// over the keys j <= position of t (causal), or all kv_lens[s] keys of t's
// sequence s, where token t of the last n = cu[s+1] - cu[s] has position
// kv_lens[s] - n + (t - cu[s]).  Query head h reads KV head h / (heads /
// kv_heads).  One pass with the running maximum and sum of the softmax in
// fp32; a row that sees no key is zero.
//
// Calls with many rows per sequence go to the tensor-core tiles of
// kv4_tiles.cu; the rest of this file is for single tokens and a few.
//
// A warp takes a tile of 4, 8 or 16 rows (the query heads of one KV head,
// token by token) and a range of the sequence's pages.  One bulk copy brings a
// page's block of the KV head (2560 G bytes) into the warp's own ring in
// shared memory; nothing else of the cache is read.  Per page, with keys and
// head dims as the 16 rows of m16n8k16 matrix instructions and 8 query rows as
// their columns (a single token has few, and the cache's side is the one that
// must be unpacked):
//   S^T = K Q^T with fp32 sums.  Codes enter as fp16 numbers by one logic
//     operation each: nibbles at bits 0..3 and 4..7 of a half are the fp16
//     subnormals n 2^-24 and n 2^-20, so two of them need no shift.  Q is
//     scaled row by row with a power of two into fp16 (and by 2^-4 more where
//     it meets the second kind), which rounds nothing that is not 2^-35 of the
//     row's largest.  The group's scale multiplies the 32-dim partial sums in
//     fp32; the offsets enter as one more matrix instruction, sum_g (16 s_g +
//     b_g) sum(q_g), with the sums of q split into two 16-bit numbers.  So a
//     score is exact but for fp32 sums and 2^-16 of that term.
//   P^T = 2^(S^T scale log2e - m), against the row's exponent offset m, which
//     is raised (and O, l rescaled) only when a score exceeds it by 2^8.  In fp16
//     P is 2^7 larger, so that weights of 2^-21 of the largest keep their bits (those
//     below 2^-32 are 0); in bf16, whose values may be as large as fp32's, it is 2^20
//     smaller, so that O stays below the largest value for 4,096 keys and more.
//   O^T += V^T P^T with V = (16 + n) s + b by one 16-bit fused multiply-add
//     per two values, rounded to T once.  P enters as two numbers of T, so its
//     rounding is left out: the error is V's rounding and the output's, 1.4
//     times that of the output's alone (1.7 with one P).  With up to 4 rows the
//     second part takes the columns that would lie idle, else instructions of
//     its own.  P^T becomes an operand by a transposition of 8 x 8.
// Where a block's warps share a row tile, they join their O, m and l in
// shared memory; where a sequence is also split over blocks, they go to the
// workspace and a second kernel joins them.
//
// Bound by instructions and their latency: about 1,050 a page and KV head for
// head_dim 128, 400 for 32, and 490 for a warp's queries and rows, half of them on
// the logic pipe (a shift or a three-input logic operation takes two cycles of a
// quarter of an SM), with 14 to 22 of 64 warps, as registers allow; 56 to 66 % of
// the issue slots are taken.
// One token, 32 heads on 8 KV heads of 128, 131,071 keys: 43.4 us, 60 % of the
// copy bandwidth.  2,048 sequences of 136 keys on average, 8 heads of 32: 43.5
// us, 32 %.
#include <cfloat>

#include "kv4_attention.cuh"

namespace cti {
namespace {

using namespace kv4;

constexpr double kLog2e = 1.4426950408889634;

// Warps of a block, and blocks of an SM: what registers allow.  The slots of a
// warp's ring hold pages, or, where those are large, a page's keys or its
// values.
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
__host__ __device__ constexpr bool halves(int G) { return G == 4; }
__host__ __device__ constexpr int slot_bytes(int G) {
  return halves(G) ? part_bytes(G) : block_bytes(G);
}
__host__ __device__ constexpr int slots(int G) { return G == 1 ? 3 : 2; }
__host__ __device__ constexpr int blocks_per_sm(int G, int NT) {
  return G == 4 ? (NT == 1 ? 4 : 2) : G == 2 ? (NT == 1 ? 4 : 3) : NT == 1 ? 6 : 4;
}
__host__ __device__ constexpr size_t smem_bytes(int G) {
  return (size_t)kWarps * slots(G) * (slot_bytes(G) + 8);
}

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  CTI_DEVICE static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Mma<__half> {
  CTI_DEVICE static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Word i of a lane's vectors of codes (i is known when the code is compiled).
template <int N>
CTI_DEVICE uint32_t word_of(const uint4 (&v)[N], int i) {
  return (i & 3) == 0 ? v[i >> 2].x : (i & 3) == 1 ? v[i >> 2].y
         : (i & 3) == 2 ? v[i >> 2].z : v[i >> 2].w;
}

// Transposes an 8 x 8 matrix of 16-bit values, two to a register.
CTI_DEVICE uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Bits 4 j .. 4 j + 3 of both halves of a K word as fp16: n 2^-24 for an even
// j, n 2^-20 for an odd one.
CTI_DEVICE uint32_t k_codes(uint32_t w, int j) {
  return (j < 2 ? w : w >> 8) & (j & 1 ? 0x00f000f0u : 0x000f000fu);
}

// ROWS: of a tile, 4, 8 or 16.
template <typename T, int G, int ROWS>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(G, (ROWS + 7) / 8))
    kv4_attention_kernel(const T* __restrict__ q, const uint8_t* __restrict__ pages, const Args a,
                         T* __restrict__ out) {
  using Y = Type16<T>;
  using M = Mma<T>;
  constexpr int D = 32 * G;
  constexpr int NT = (ROWS + 7) / 8;  // tiles of 8 columns
  // With 4 rows the other 4 columns are the same rows again, for the second
  // part of P.
  constexpr bool kDup = ROWS == 4;
  constexpr int S = slots(G);
  constexpr int W = kWarps;
  constexpr int kSlot = slot_bytes(G);
  constexpr float kOffUnit = Y::kShift == 3 ? 1.0f : 0x1p14f;
  constexpr float kPUnit = Y::kShift == 3 ? -20.0f : kPUnitFp16;  // of weights of 1
  constexpr int H = halves(G) ? 2 : 1;  // slots that a page takes
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = warp_id(), lane = lane_id();
  const int r8 = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + (size_t)warp * S * kSlot;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)W * S * kSlot) + warp * S;
  if (lane == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  grid_dependency_wait();

  const bool shared = a.shared != 0;
  const unsigned unit = shared ? blockIdx.x : blockIdx.x * W + warp;
  if (unit >= (unsigned)a.num_seqs * a.kv_heads) return;  // all warps of a tile alike
  const int s = (int)a.by_kv_heads(unit), kvh = (int)unit - s * a.kv_heads;
  const int group = a.group;
  const int begin = __ldg(a.cu + s), end = __ldg(a.cu + s + 1);
  const int len = __ldg(a.kv_lens + s);
  if (begin < 0 || end > a.tokens || end < begin) {
    if (lane == 0) raise_status(a.status, CTI_ERR_INVALID_ARG, s);
    if (gridDim.z > 1 && blockIdx.z == 0 && blockIdx.y == 0)
      refuse_rows(a.ws_ml, max(begin, 0), min(end, a.tokens), a.heads, group, kvh);
    return;
  }
  const int n_new = end - begin;
  const int first = max(len, 0) - n_new;  // position of the first new token
  const int rows = n_new * group;         // tokens * heads is below 2^31
  int limit = max(len, 0);                // keys that the table reaches
  if (limit > a.table_cols * kPage || (limit > 0 && a.num_pages <= 0)) {
    if (lane == 0 && rows > 0) raise_status(a.status, CTI_ERR_BOUNDS, s);
    limit = a.num_pages <= 0 ? 0 : a.table_cols * kPage;
  }
  const int32_t* table = a.table + s * a.table_stride;
  const uint8_t* base = pages + (int64_t)kvh * block_bytes(G);
  const int64_t page_stride = (int64_t)a.kv_heads * block_bytes(G);
  uint32_t count = 0;  // slots filled so far: place and parity
  bool dead = false;   // a copy did not arrive in time

  for (int tile = blockIdx.y; tile < (rows + ROWS - 1) / ROWS; tile += gridDim.y) {
    // Keys that some row and that every row of the tile sees.
    const int row0 = tile * ROWS, row_last = min(rows, row0 + ROWS) - 1;
    const int most =
        max(a.causal ? min(first + (int)a.by_group(row_last) + 1, limit) : limit, 0);
    const int all = a.causal ? min(first + (int)a.by_group(row0) + 1, limit) : limit;

    // ---- this warp's pages ----
    int p0 = 0, np = (most + kPage - 1) / kPage;
    if (gridDim.z > 1) {  // the last block takes what the caller's bound left out
      p0 = min(np, (int)blockIdx.z * a.chunk);
      np = (blockIdx.z == gridDim.z - 1 ? np : min(np, p0 + a.chunk)) - p0;
    }
    if (shared) {
      const int per = (np + W - 1) / W, skip = min(np, warp * per);
      p0 += skip;
      np = min(np - skip, per);
    }
    if (dead) np = 0;
    int ids = -1;      // lane i: page p0 + (chunk of 32) + i
    uint32_t bad[2] = {0, 0};  // by chunk: bit per page that is none; nothing of it is seen
    auto issue = [&](int h) {  // page i of the range; with halves its keys (h = 2 i) or values
      const int i = h / H;
      if ((h & (32 * H - 1)) == 0) {
        ids = i + lane < np ? __ldg(table + p0 + i + lane) : 0;
        if (ids < 0 || ids >= a.num_pages) {
          raise_status(a.status, CTI_ERR_BOUNDS, s);
          ids = -1;
        }
        bad[(i >> 5) & 1] = __ballot_sync(0xffffffffu, ids < 0);
      }
      const int id = __shfl_sync(0xffffffffu, ids, i & 31);
      const uint32_t slot = (count + h) % S;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[slot], kSlot);
        bulk_load(ring + slot * kSlot, base + max(id, 0) * page_stride + (h & (H - 1)) * kSlot,
                  kSlot, &full[slot]);
      }
    };
    auto arrived = [&](int h) {
      return __all_sync(0xffffffffu, mbar_wait(&full[(count + h) % S], ((count + h) / S) & 1,
                                               a.status, 0x700, nullptr));
    };
#pragma unroll 1
    for (int h = 0; h < S && h < H * np; ++h) issue(h);

    // ---- queries: lane 4 r + t has dims 8 t .. + 7 of every group of row r ----
    uint32_t qb[NT][G][4];
    uint32_t off_b[NT][2];
    float sl[NT][2];  // of rows 2 t and 2 t + 1, for scores in units of the row's scale
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + 8 * n + (kDup ? r8 & 3 : r8);
      const int i = (int)a.by_group(row), h = kvh * group + row - i * group;
      uint4 v[G];
      float most_q = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        v[g] = make_uint4(0, 0, 0, 0);
        if (row < rows)
          v[g] = __ldg(reinterpret_cast<const uint4*>(q + (begin + i) * a.q_stride +
                                                      (int64_t)h * D + 32 * g + 8 * t4));
        const uint32_t w[4] = {v[g].x, v[g].y, v[g].z, v[g].w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          most_q = fmaxf(most_q, fmaxf(fabsf(Y::low(w[j])), fabsf(Y::high(w[j]))));
      }
      most_q = fmaxf(most_q, __shfl_xor_sync(0xffffffffu, most_q, 1));
      most_q = fmaxf(most_q, __shfl_xor_sync(0xffffffffu, most_q, 2));
      const int k = query_exponent(most_q, a);
      const float up = power_of_two(k) * a.sign;
      float sum_mine = 0.0f;  // of group t4's 32 dims (G = 2: t4 & 1; G = 1: the only one)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint32_t w[4] = {v[g].x, v[g].y, v[g].z, v[g].w};
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = Y::low(w[j]) * up, y = Y::high(w[j]) * up;
          sum += x + y;
          const float f = j & 1 ? 0.0625f : 1.0f;
          qb[n][g][j] = Type16<__half>::pack(x * f, y * f);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (g == (t4 & (G - 1))) sum_mine = sum;
      }
      // The offsets' operand: the rows that meet s and b of a group are 16 and
      // 1 times the sum of q in it, in two parts, in the scores' units (fp16
      // cannot hold those: 2^14 above them).
      sum_mine *= kOffUnit * 0x1p-24f;
      const float hi = Y::to_float(Y::bits(sum_mine));
      const float lo = sum_mine - hi;
      const uint32_t hi2 = Y::pack(16.0f * hi, hi), lo2 = Y::pack(16.0f * lo, lo);
      off_b[n][0] = G == 4 || t4 < G ? hi2 : t4 < 2 * G ? lo2 : 0u;
      off_b[n][1] = G == 4 ? lo2 : 0u;
      const float mine = a.scale_m * power_of_two(min(a.scale_e + 24 - k, 128));
      sl[n][0] = __shfl_sync(0xffffffffu, mine, 8 * t4);
      sl[n][1] = __shfl_sync(0xffffffffu, mine, 8 * t4 + 4);
    }
    int sees[NT][2];  // keys that rows 2 t and 2 t + 1 see
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = min(row0 + 8 * n + (kDup ? 2 * t4 & 3 : 2 * t4) + e, row_last);
        sees[n][e] = a.causal ? min(first + (int)a.by_group(row) + 1, limit) : limit;
      }

    float o[NT][2 * G][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2 * G; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
    }

    const uint64_t part_x = t4 < 2 ? 0 : f2_pack(1.0f, 1.0f);
    const uint64_t part_top = t4 < 2 ? f2_pack(1.0f, 1.0f) : f2_pack(-1.0f, -1.0f);

    int done = 0;
    for (; done < np; ++done) {
      if (!arrived(H * done)) break;
      uint8_t* blk = ring + (count + H * done) % S * kSlot;
      uint8_t* vblk = H == 1 ? blk + part_bytes(G) : ring + (count + 2 * done + 1) % S * kSlot;

      // ---- S^T = K Q^T, 16 keys at a time ----
      float sc[NT][4][4];
      uint4 kw[2];  // of 16 tokens (G = 4), 32 (2) or 64 (1)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        constexpr int kTiles = 4 / G;  // of 16 tokens, that the two vectors hold
        if (mt % kTiles == 0) {
#pragma unroll
          for (int v = 0; v < 2; ++v)
            kw[v] = *reinterpret_cast<const uint4*>(
                blk + ((2 * (mt / kTiles) + v) * 32 + lane) * 16);
        }
        uint32_t meta[2][G];  // of tokens 16 mt + r and + 8
        uint32_t am[2];       // its word for the offsets: group t's
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t* mw =
              reinterpret_cast<const uint32_t*>(blk + k_meta_at(G)) + (16 * mt + 8 * e + r8) * G;
          if constexpr (G == 4) {
            const uint4 y = *reinterpret_cast<const uint4*>(mw);
            meta[e][0] = y.x, meta[e][1] = y.y, meta[e][2] = y.z, meta[e][3] = y.w;
          } else if constexpr (G == 2) {
            const uint2 y = *reinterpret_cast<const uint2*>(mw);
            meta[e][0] = y.x, meta[e][1] = y.y;
          } else {
            meta[e][0] = *mw;
          }
          am[e] = G == 1 ? meta[e][0] : mw[t4 & (G - 1)];
        }
        const uint32_t off_a[4] = {am[0], am[1], G == 4 ? am[0] : 0u, G == 4 ? am[1] : 0u};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[n][mt][e] = 0.0f;
          Mma<T>::run(sc[n][mt], off_a, off_b[n][0], off_b[n][1]);
          if (kOffUnit != 1.0f) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][mt][e] *= 1.0f / kOffUnit;
          }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t w0 = word_of(kw, 2 * (mt % kTiles) * G + g);
          const uint32_t w1 = word_of(kw, (2 * (mt % kTiles) + 1) * G + g);
          const uint32_t a0[4] = {k_codes(w0, 0), k_codes(w1, 0), k_codes(w0, 1), k_codes(w1, 1)};
          const uint32_t a1[4] = {k_codes(w0, 2), k_codes(w1, 2), k_codes(w0, 3), k_codes(w1, 3)};
          const float s0 = Y::low(meta[0][g]), s1 = Y::low(meta[1][g]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            Mma<__half>::run(c, a0, qb[n][g][0], qb[n][g][1]);
            Mma<__half>::run(c, a1, qb[n][g][2], qb[n][g][3]);
            float(&x)[4] = sc[n][mt];
            f2_unpack(f2_fma(f2_pack(c[0], c[1]), f2_pack(s0, s0), f2_pack(x[0], x[1])), x[0],
                      x[1]);
            f2_unpack(f2_fma(f2_pack(c[2], c[3]), f2_pack(s1, s1), f2_pack(x[2], x[3])), x[2],
                      x[3]);
          }
        }
      }

      if (H == 2) {
        __syncwarp();
        if (2 * done + S < 2 * np) issue(2 * done + S);
        if (!arrived(2 * done + 1)) break;
      }

      const int key0 = (p0 + done) * kPage;
      const bool is_bad = bad[(done >> 5) & 1] >> (done & 31) & 1;
      if (is_bad || key0 + kPage > all) {
        // Keys that a row does not see count nothing, whatever they hold: a
        // value behind the last key gets a meta of zero.  One that is not
        // finite and that only some rows see gets the same, and a score of NaN
        // for those that do.
        const int lim_most = is_bad ? 0 : most - key0;
        uint32_t* vm =
            reinterpret_cast<uint32_t*>(vblk + v_meta_at(G) - v_codes_at(G)) + lane * 2 * G;
        bool nan0 = false, nan1 = false;  // of tokens 2 lane and 2 lane + 1
        if (all < most) {
#pragma unroll
          for (int i = 0; i < 2 * G; ++i) {
            nan0 |= (vm[i] & Inf16<T>::kBits) == Inf16<T>::kBits;
            nan1 |= ((vm[i] >> 16) & Inf16<T>::kBits) == Inf16<T>::kBits;
          }
        }
        const uint32_t keep = (nan0 || 2 * lane >= lim_most ? 0u : 0xffffu) |
                              (nan1 || 2 * lane + 1 >= lim_most ? 0u : 0xffff0000u);
        if (keep != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 2 * G; ++i) vm[i] &= keep;
        }
        const uint32_t even = __ballot_sync(0xffffffffu, nan0);
        const uint32_t odd = __ballot_sync(0xffffffffu, nan1);
        if (even | odd) {
          const uint32_t mine = r8 & 1 ? odd : even;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
              if (mine >> (8 * mt + (r8 >> 1)) & 1) sc[n][mt][0] = sc[n][mt][1] = NAN;
              if (mine >> (8 * mt + 4 + (r8 >> 1)) & 1) sc[n][mt][2] = sc[n][mt][3] = NAN;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int lim0 = (is_bad ? 0 : sees[n][0] - key0) - r8;
          const int lim1 = (is_bad ? 0 : sees[n][1] - key0) - r8;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            if (16 * mt >= lim0) sc[n][mt][0] = -INFINITY;
            if (16 * mt >= lim1) sc[n][mt][1] = -INFINITY;
            if (16 * mt + 8 >= lim0) sc[n][mt][2] = -INFINITY;
            if (16 * mt + 8 >= lim1) sc[n][mt][3] = -INFINITY;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
      }

      // ---- the rows' exponent offsets ----
      float mx[NT][2];
      bool raise = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(sc[n][0][e], sc[n][0][2 + e]);
#pragma unroll
          for (int mt = 1; mt < 4; ++mt) x = max3f(x, sc[n][mt][e], sc[n][mt][2 + e]);
          mx[n][e] = x;
          raise = raise || (x - m[n][e]) * sl[n][e] > kSlack;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = mx[n][e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            if (x > m[n][e]) {
              const float corr = ex2_approx((m[n][e] - x) * sl[n][e]);
              m[n][e] = x;
              l[n][e] *= corr;
#pragma unroll
              for (int i = 0; i < 2 * G; ++i) {
                o[n][i][e] *= corr;
                o[n][i][2 + e] *= corr;
              }
            }
          }
      }

      // ---- P^T, and O^T += V^T P^T, 16 keys at a time ----
      float noff[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          noff[n][e] = m[n][e] == -INFINITY ? 0.0f : fmaf(-m[n][e], sl[n][e], kPUnit);
      uint4 vw[2];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        constexpr int kTiles = 4 / G;
        if (kk % kTiles == 0) {
#pragma unroll
          for (int v = 0; v < 2; ++v)
            vw[v] = *reinterpret_cast<const uint4*>(
                vblk + ((2 * (kk / kTiles) + v) * 32 + lane) * 16);
        }
        uint32_t pb[NT][2], pl[NT][2];  // P^T, and what its rounding left
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float(&x)[4] = sc[n][kk];
          const uint64_t sl2 = f2_pack(sl[n][0], sl[n][1]), no2 = f2_pack(noff[n][0], noff[n][1]);
          f2_unpack(f2_fma(f2_pack(x[0], x[1]), sl2, no2), x[0], x[1]);
          f2_unpack(f2_fma(f2_pack(x[2], x[3]), sl2, no2), x[2], x[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = ex2_approx(x[e]);
          f2_unpack(f2_add(f2_pack(l[n][0], l[n][1]),
                           f2_add(f2_pack(x[0], x[1]), f2_pack(x[2], x[3]))),
                    l[n][0], l[n][1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (kDup) {
              // The upper bits of p in columns 0..3, the rest in 4..7.
              const uint64_t top = f2_pack(
                  __uint_as_float(__float_as_uint(x[2 * e]) & Y::kTopBits),
                  __uint_as_float(__float_as_uint(x[2 * e + 1]) & Y::kTopBits));
              float y0, y1;
              f2_unpack(f2_fma(f2_pack(x[2 * e], x[2 * e + 1]), part_x, f2_mul(top, part_top)),
                        y0, y1);
              pb[n][e] = transpose8(Y::pack(y0, y1));
            } else {
              const uint32_t p = Y::pack(x[2 * e], x[2 * e + 1]);
              pb[n][e] = transpose8(p);
              pl[n][e] = transpose8(Y::pack(x[2 * e] - Y::low(p), x[2 * e + 1] - Y::high(p)));
            }
          }
        }
        uint2 meta[2][G];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint2* mw =
              reinterpret_cast<const uint2*>(vblk + v_meta_at(G) - v_codes_at(G)) +
              (8 * kk + 4 * e + t4) * G;
          if constexpr (G == 1) {
            meta[e][0] = *mw;
          } else {
#pragma unroll
            for (int g = 0; g < G; g += 2) {
              const uint4 y = *reinterpret_cast<const uint4*>(mw + g);
              meta[e][g] = make_uint2(y.x, y.y);
              meta[e][g + 1] = make_uint2(y.z, y.w);
            }
          }
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t w0 = word_of(vw, 2 * (kk % kTiles) * G + g);
          const uint32_t w1 = word_of(vw, (2 * (kk % kTiles) + 1) * G + g);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t av[4] = {
                fma2<T>(code_pair<T>(w0, 2 * j), meta[0][g].x, meta[0][g].y),
                fma2<T>(code_pair<T>(w0, 2 * j + 1), meta[0][g].x, meta[0][g].y),
                fma2<T>(code_pair<T>(w1, 2 * j), meta[1][g].x, meta[1][g].y),
                fma2<T>(code_pair<T>(w1, 2 * j + 1), meta[1][g].x, meta[1][g].y)};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              M::run(o[n][2 * g + j], av, pb[n][0], pb[n][1]);
              if (!kDup) M::run(o[n][2 * g + j], av, pl[n][0], pl[n][1]);
            }
          }
        }
      }
      __syncwarp();
      if (H * (done + 1) - 1 + S < H * np) issue(H * (done + 1) - 1 + S);
    }
    if (done < np) {  // let the copies in flight land, then give up
      dead = true;
      for (int h = H * done; h < H * np && h <= H * done + S; ++h) arrived(h);
    }
    count += H * np;

    // ---- join and store: lane 4 r + t has dims 4 r .. + 3 of every group ----
    if (kDup) {
#pragma unroll
      for (int i = 0; i < 2 * G; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][i][e] += __shfl_xor_sync(0xffffffffu, o[0][i][e], 2);
    }
    const bool holds = !kDup || t4 < 2;  // rows of its own
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
        l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
      }
    if (shared) {
      // Every warp's rows in its own ring, then the first warp adds them up.
      float* mine = reinterpret_cast<float*>(ring);
      static_assert((ROWS * D + 2 * ROWS) * 4 <= S * kSlot, "room for the rows");
      __syncwarp();
      if (warp != 0 && holds) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = 8 * n + 2 * t4 + e;
#pragma unroll
            for (int g = 0; g < G; ++g)
              *reinterpret_cast<float4*>(mine + row * D + 32 * g + 4 * r8) =
                  make_float4(o[n][2 * g][e], o[n][2 * g][2 + e], o[n][2 * g + 1][e],
                              o[n][2 * g + 1][2 + e]);
            if (r8 == 0)
              *reinterpret_cast<float2*>(mine + ROWS * D + 2 * row) =
                  make_float2(m[n][e], l[n][e]);
          }
      }
      __syncthreads();
      if (warp == 0 && holds) {
        for (int w = 1; w < W; ++w) {
          const float* src = reinterpret_cast<const float*>(ring + (size_t)w * S * kSlot);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = 8 * n + 2 * t4 + e;
              const float2 ml = *reinterpret_cast<const float2*>(src + ROWS * D + 2 * row);
              const float mm = fmaxf(m[n][e], ml.x);
              const float ca = m[n][e] == mm ? 1.0f : ex2_approx((m[n][e] - mm) * sl[n][e]);
              const float cb = ml.x == mm ? 1.0f : ex2_approx((ml.x - mm) * sl[n][e]);
              m[n][e] = mm;
              l[n][e] = l[n][e] * ca + ml.y * cb;
#pragma unroll
              for (int g = 0; g < G; ++g) {
                const float4 x =
                    *reinterpret_cast<const float4*>(src + row * D + 32 * g + 4 * r8);
                o[n][2 * g][e] = o[n][2 * g][e] * ca + x.x * cb;
                o[n][2 * g][2 + e] = o[n][2 * g][2 + e] * ca + x.y * cb;
                o[n][2 * g + 1][e] = o[n][2 * g + 1][e] * ca + x.z * cb;
                o[n][2 * g + 1][2 + e] = o[n][2 * g + 1][2 + e] * ca + x.w * cb;
              }
            }
        }
      }
    }
    if ((!shared || warp == 0) && holds) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = row0 + 8 * n + 2 * t4 + e;
          if (row >= rows) continue;
          const int i = (int)a.by_group(row);
          const int64_t at = (int64_t)(begin + i) * a.heads + kvh * group + row - i * group;
          const float inv = l[n][e] == 0.0f ? 0.0f : 1.0f / l[n][e];
          if (gridDim.z == 1) {
#pragma unroll
            for (int g = 0; g < G; ++g)
              *reinterpret_cast<uint2*>(out + at * D + 32 * g + 4 * r8) =
                  make_uint2(Y::pack(o[n][2 * g][e] * inv, o[n][2 * g][2 + e] * inv),
                             Y::pack(o[n][2 * g + 1][e] * inv, o[n][2 * g + 1][2 + e] * inv));
          } else {
            const int64_t ws = (int64_t)blockIdx.z * a.tokens * a.heads + at;
            // m times its row's scale: a power of 2 that weights can be told by
            if (r8 == 0)
              a.ws_ml[ws] = make_float2(m[n][e] == -INFINITY ? -INFINITY : m[n][e] * sl[n][e],
                                        l[n][e]);
            if (np > 0) {  // else the block has no pages (the first warp's come first)
#pragma unroll
              for (int g = 0; g < G; ++g)
                *reinterpret_cast<float4*>(a.ws_o + ws * D + 32 * g + 4 * r8) =
                    make_float4(o[n][2 * g][e] * inv, o[n][2 * g][2 + e] * inv,
                                o[n][2 * g + 1][e] * inv, o[n][2 * g + 1][2 + e] * inv);
            }
          }
        }
    }
    if (shared) {
      // The rings are free again (copies may overwrite them) once the first
      // warp has read them.
      fence_proxy_async_smem();
      __syncthreads();
    }
  }
}

// Joins the splits of every row, each with its own O / l, m and l: a block per
// row, whose warps share the splits.
// Bound by latency (the rows of a call with splits are few): every warp finds
// all weights, 32 splits at a time, then sums its own splits with independent
// loads.
constexpr int kJoinWarps = 4;
template <typename T, int G>
__global__ void __launch_bounds__(kJoinWarps * 32)
    kv4_join_kernel(const Args a, int splits, T* __restrict__ out) {
  using Y = Type16<T>;
  constexpr int D = 32 * G;
  __shared__ float part[kJoinWarps][D];
  grid_dependency_wait();
  const int64_t rows = (int64_t)a.tokens * a.heads, row = blockIdx.x;
  const int lane = lane_id(), warp = warp_id();
  const int t = blockIdx.x / (unsigned)a.heads;
  if (t < __ldg(a.cu) || t >= __ldg(a.cu + a.num_seqs)) return;
  float2 ml[4];  // of splits 32 i + lane
  float mm = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ml[i] = make_float2(-INFINITY, 0.0f);
    if (32 * i + lane < splits) ml[i] = a.ws_ml[(32 * i + lane) * rows + row];
    mm = fmaxf(mm, ml[i].x);
  }
  if (__shfl_sync(0xffffffffu, ml[0].y, 0) < 0.0f) return;  // a refused sequence's
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
  float l = 0.0f, o[G], w[4];
#pragma unroll
  for (int g = 0; g < G; ++g) o[g] = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // No key of the split is seen where l is 0: its rows were not written.
    w[i] = ml[i].y == 0.0f ? 0.0f : ml[i].y * (ml[i].x == mm ? 1.0f : ex2_approx(ml[i].x - mm));
    l += w[i];
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  // Weights that add up to 1, so that the sum does not pass the largest value.
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (32 * i >= splits) break;
#pragma unroll 8
    for (int z = warp; z < min(32, splits - 32 * i); z += kJoinWarps) {
      const float wz = __shfl_sync(0xffffffffu, w[i] * inv, z);
      if (wz == 0.0f) continue;
      const float* src = a.ws_o + ((32 * i + z) * rows + row) * D + lane;
#pragma unroll
      for (int g = 0; g < G; ++g) o[g] = fmaf(src[32 * g], wz, o[g]);
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) part[warp][32 * g + lane] = o[g];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += kJoinWarps * 32) {
    float sum = part[0][d];
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) sum += part[w][d];
    reinterpret_cast<uint16_t*>(out)[row * D + d] = (uint16_t)Y::bits(sum);
  }
}

// Query rows of a KV head, by the caller's bound, from which a sequence's rows
// are taken in tiles of 128 on the tensor cores: the first where the sequences' KV
// heads fill half of the GPU, else the second.  Measured, us here and there, 2,000
// keys, head_dim 32 / 64 / 128:
//   96 sequences of 4 KV heads: 64 rows, 72 and 80 / 104 and 100 / 180 and 164;
//                               96 rows, 98 and 80 / 145 and 100 / 254 and 166
//   8 sequences:                64 rows, 20 and 22 / 24 and 24 / 32 and 34;
//                              128 rows, 26 and 24 / 38 and 26 / 48 and 38
//   1 sequence of 8 KV heads:  128 rows, 17 and 20 / 17 and 24 / 22 and 34
// That is bf16; fp16's tiles take a tenth to a third longer, and are ahead from 80
// rows on.
constexpr int kTilesFrom = 65, kTilesFromFew = 97;

// Bytes that the splits' outputs may take.  Calls that would need more have rows
// enough to fill the GPU without so many splits.
constexpr int64_t kWorkspaceMost = (int64_t)64 << 20;

// How a call is laid out over the GPU; a function of the sizes alone.
struct Plan {
  int big;             // 128-row tiles of a block (kv4_tiles.cu), 1 or 2; 0: warps as here
  int rows;            // that a warp takes: 4, 8 or 16
  bool shared;         // a block's warps share a tile's pages
  int splits, chunk;   // blocks that share them, and the pages of each
  int64_t tiles;       // row tiles of a sequence
};

Plan plan(int num_seqs, int64_t tokens, int max_new, int64_t max_kv_len, int heads, int kv_heads,
          int head_dim) {
  const int G = head_dim / kGroup;
  const int64_t most = max_new < tokens ? max_new : tokens;
  const int64_t rows = (most > 0 ? most : 1) * (heads / kv_heads);
  // No table reaches further, whatever the bound: pages, and a split's first, are ints.
  const int64_t len = max_kv_len < INT32_MAX ? max_kv_len : INT32_MAX;
  const int64_t pages = len > 0 ? (len + kPage - 1) / kPage : 1;
  Plan p = {};
  const double sequences = (double)num_seqs * kv_heads;
  const int64_t split_bytes = tokens * heads * (head_dim * (int64_t)sizeof(float) +
                                                (int64_t)sizeof(float2));
  int64_t most_splits = (kWorkspaceMost - 512) / split_bytes;  // but for alignment
  most_splits = most_splits < 1 ? 1 : most_splits > 128 ? 128 : most_splits;
  if (rows >= (sequences >= kSMs / 2 ? kTilesFrom : kTilesFromFew)) {
    // Two tiles share the unpacking of a page, which costs less than one of two
    // blocks' latency hidden by the other, but for head_dim 32 (2,048 rows of 384
    // KV heads over 2,000 keys: 1092 us with two, 1071 with one; for 64, 1235 and
    // 1378; for 128, 1639 and 2264; 192 rows: 133 and 131, 150 and 168, 197 and
    // 268).  Fewer blocks than the GPU holds share the pages, eight at least.
    p.big = rows > 128 && G > 1 ? 2 : 1;
    p.tiles = (rows + 128 * p.big - 1) / (128 * p.big);
    const double blocks = sequences * (double)p.tiles;
    int64_t splits = (int64_t)(kSMs * (3 - p.big) / blocks);
    splits = splits > pages / 8 ? pages / 8 : splits;
    p.splits = (int)(splits < 1 ? 1 : splits > most_splits ? most_splits : splits);
    p.chunk = (int)((pages + p.splits - 1) / p.splits);
    return p;
  }
  // (96 sequences of 4 KV heads, 2,000 keys, head_dim 32 / 64 / 128: 8 rows in
  // tiles of 4 33 us / 39 / 64, of 8 25 / 31 / 45; 16 rows in tiles of 8 35 / 41 /
  // 68, of 16 35 / 43 / 59; 48 rows 66 / 92 / 162, 53 / 80 / 133, and, for 32 and
  // 64, 72 / 102 in tiles of 32.)
  p.rows = rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
  p.tiles = (rows + p.rows - 1) / p.rows;
  const double units = sequences * (double)p.tiles;
  const double room = (double)kSMs * blocks_per_sm(G, (p.rows + 7) / 8) * kWarps;  // warps at once
  p.splits = 1;
  p.chunk = 0;
  if (units >= room && pages <= (units >= 4 * room ? 64 : 16)) {
    // More tiles than warps, and none so long that the last ones run alone: a
    // warp each.  (Lengths up to 16 pages, 8 heads of 32: 600 sequences 82 us,
    // 92 shared; 2,400 sequences 135 and 170.  Up to 64 pages: 300 sequences,
    // less than four times the warps, 158 and 140; 2,400 sequences 446 and 511.)
    p.shared = false;
    return p;
  }
  // A block's warps share a tile; with long sequences, blocks do too, so that
  // all run at once, or, where that is more than 16 pages for a warp, in
  // pieces of 12, small enough that sequences of any lengths balance out (48
  // sequences of 1,000 to 8,000 keys, 8 KV heads of 128: 81 us, 91 without and 85
  // with pieces of 4; 128 of 100 to 16,000: 294, 335 and 343).
  p.shared = true;
  const double ideal = units * pages / room;
  int64_t per_warp = ideal > 16 ? 12 : (int64_t)ideal + 1;
  p.chunk = (int)(per_warp * kWarps);
  int64_t splits = (pages + p.chunk - 1) / p.chunk;
  if (splits > most_splits) {
    splits = most_splits;
    p.chunk = (int)((pages + splits - 1) / splits);
  }
  p.splits = (int)splits;
  return p;
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

size_t workspace_o_bytes(const Plan& p, int64_t tokens, int heads, int head_dim) {
  return p.splits > 1 ? align256((size_t)p.splits * tokens * heads * head_dim * sizeof(float)) : 0;
}

template <typename T, int G, int ROWS>
int launch(const void* q, const void* pages, const Args& a, const Plan& p, void* out,
           cudaStream_t s) {
  static uint64_t configured = 0;
  if (ensure_smem_limit(kv4_attention_kernel<T, G, ROWS>, (int)smem_bytes(G), configured) !=
      cudaSuccess)
    return CTI_ERR_CUDA;
  const int64_t units = (int64_t)a.num_seqs * a.kv_heads;
  const int per = p.shared ? 1 : kWarps;
  const dim3 grid((unsigned)((units + per - 1) / per),
                  (unsigned)(p.tiles < 65535 ? p.tiles : 65535), (unsigned)p.splits);
  if (launch_dependent(kv4_attention_kernel<T, G, ROWS>, grid, dim3(kThreads), smem_bytes(G), s,
                       static_cast<const T*>(q), static_cast<const uint8_t*>(pages), a,
                       static_cast<T*>(out)) != cudaSuccess)
    return CTI_ERR_CUDA;
  return CTI_OK;
}

template <typename T, int G>
int launch_join(const Args& a, int splits, void* out, cudaStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.tokens * a.heads));
  return launch_dependent(kv4_join_kernel<T, G>, grid, dim3(kJoinWarps * 32), 0, s, a, splits,
                          static_cast<T*>(out)) == cudaSuccess
             ? CTI_OK
             : CTI_ERR_CUDA;
}

template <typename T, int G>
int launch_shape(const void* q, const void* pages, const Args& a, const Plan& p, int dtype,
                 void* out, cudaStream_t s) {
  int rc;
  if (p.big) {
    rc = launch_tiles(q, pages, a, dtype, 32 * G, p.big, p.tiles, p.splits, out, s);
  } else if (p.rows == 4) {
    rc = launch<T, G, 4>(q, pages, a, p, out, s);
  } else if (p.rows == 8) {
    rc = launch<T, G, 8>(q, pages, a, p, out, s);
  } else {
    rc = launch<T, G, 16>(q, pages, a, p, out, s);
  }
  if (rc != CTI_OK || p.splits == 1) return rc;
  return launch_join<T, G>(a, p.splits, out, s);
}

template <typename T>
int launch_dim(const void* q, const void* pages, const Args& a, const Plan& p, int dtype,
               int head_dim, void* out, cudaStream_t s) {
  return head_dim == 32   ? launch_shape<T, 1>(q, pages, a, p, dtype, out, s)
         : head_dim == 64 ? launch_shape<T, 2>(q, pages, a, p, dtype, out, s)
                          : launch_shape<T, 4>(q, pages, a, p, dtype, out, s);
}

}  // namespace
}  // namespace cti

extern "C" size_t cti_kv4_attention_workspace_bytes(int num_seqs, int64_t tokens, int max_new,
                                                    int64_t max_kv_len, int heads, int kv_heads,
                                                    int head_dim) {
  using namespace cti;
  if (num_seqs <= 0 || tokens <= 0 || max_kv_len < 0 || heads <= 0 || kv_heads <= 0 ||
      heads % kv_heads != 0 || (head_dim != 32 && head_dim != 64 && head_dim != 128))
    return 0;
  const Plan p = plan(num_seqs, tokens, max_new, max_kv_len, heads, kv_heads, head_dim);
  const size_t o = workspace_o_bytes(p, tokens, heads, head_dim);
  return o ? o + align256((size_t)p.splits * tokens * heads * sizeof(float2)) : 0;
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
  if (tokens > INT32_MAX - 256 || heads > 65535 || tokens * heads > INT32_MAX - 512 ||
      (int64_t)num_seqs * kv_heads > INT32_MAX || table_cols > INT32_MAX / kv4::kPage)
    return CTI_ERR_UNSUPPORTED;
  if (num_seqs == 0 || tokens == 0) return CTI_OK;
  if (!q || !out || !pages || !cu_seqlens || !kv_lens || (!page_table && table_cols > 0))
    return CTI_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(out) || !aligned16(pages)) return CTI_ERR_INVALID_ARG;
  if (q_stride % 8 != 0 || q_stride < (int64_t)heads * head_dim || table_stride < table_cols)
    return CTI_ERR_INVALID_ARG;
  const Plan p = plan(num_seqs, tokens, max_new, max_kv_len, heads, kv_heads, head_dim);
  const size_t ws_o = workspace_o_bytes(p, tokens, heads, head_dim);
  if (ws_o &&
      (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0 ||
       workspace_bytes < cti_kv4_attention_workspace_bytes(num_seqs, tokens, max_new, max_kv_len,
                                                           heads, kv_heads, head_dim)))
    return CTI_ERR_INVALID_ARG;
  int scale_e = 0;
  const double scale_m = scale == 0.0f ? 1.0 : frexp(fabs((double)scale) * kLog2e, &scale_e);
  const Args a = {cu_seqlens,
                  kv_lens,
                  page_table,
                  table_stride,
                  table_cols,
                  num_seqs,
                  (int)tokens,
                  heads,
                  kv_heads,
                  heads / kv_heads,
                  (float)scale_m,
                  scale_e,
                  scale == 0.0f ? 0.0f : copysignf(1.0f, scale),
                  causal,
                  num_pages,
                  q_stride,
                  Divisor((uint32_t)(heads / kv_heads)),
                  Divisor((uint32_t)kv_heads),
                  p.shared,
                  p.chunk,
                  static_cast<float*>(workspace),
                  reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + ws_o),
                  status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == CTI_DTYPE_BF16
             ? launch_dim<__nv_bfloat16>(q, pages, a, p, dtype, head_dim, out, s)
             : launch_dim<__half>(q, pages, a, p, dtype, head_dim, out, s);
}
