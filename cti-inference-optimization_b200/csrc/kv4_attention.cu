// Attention of new tokens over the 4-bit key/value cache (format: kv4.cuh):
//   out[t, h, :] = sum_j softmax_j(scale q[t, h, :] . k_j) v_j
// over the keys j <= position of t (causal), or all kv_lens[s] keys of t's
// sequence s, where token t of the last n = cu[s+1] - cu[s] has position
// kv_lens[s] - n + (t - cu[s]).  Query head h reads KV head h / (heads /
// kv_heads).  One pass with the running maximum and sum of the softmax in
// fp32; a row that sees no key is zero.
//
// A warp takes a tile of up to 16 rows (the query heads of one KV head, token
// by token) and a range of the sequence's pages.  One bulk copy brings a
// page's block of the KV head (2560 G bytes) into the warp's own ring in
// shared memory; nothing else of the cache is read.  Per page:
//   S = Q K^T by m16n8k16 matrix instructions with fp32 sums.  A code n is
//     turned into the 16-bit number 16 + n by a shift and a logic operation,
//     exactly; the group's scale multiplies the 32-dim partial sums in fp32,
//     and the bases enter as one more matrix instruction, sum_g b_g sum(q_g),
//     with the sums of q split into two 16-bit numbers.  So a score is exact
//     but for fp32 sums and 2^-16 of that term.
//   P = 2^(S scale log2e - m), against the row's exponent offset m, which is
//     raised (and O, l rescaled) only when a score exceeds it by 2^8.
//   O += P V with V = (16 + n) s + b by one 16-bit fused multiply-add per two
//     values; P and V are rounded to 16 bits once each, as 16-bit attention
//     does.
// The warps of a row tile (1, 2 or 4 of a block) join their O, m and l in
// shared memory; where a sequence is also split over blocks, they go to the
// workspace and a second kernel joins them.
#include <cfloat>

#include "kv4.cuh"

namespace cti {
namespace {

using namespace kv4;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kSMs = 148;
constexpr float kSlack = 8.0f;
constexpr float kLog2e = 1.4426950408889634f;

__host__ __device__ constexpr int stages(int G) { return G == 1 ? 4 : G == 2 ? 3 : 2; }
__host__ __device__ constexpr int blocks_per_sm(int G) { return G == 1 ? 4 : G == 2 ? 3 : 2; }
__host__ __device__ constexpr size_t smem_bytes(int G) {
  return (size_t)kWarps * stages(G) * block_bytes(G) + kWarps * stages(G) * 8;
}

struct Args {
  const int32_t* cu;
  const int32_t* kv_lens;
  const int32_t* table;
  int64_t table_stride;
  int table_cols;
  int num_seqs;
  int tokens;
  int heads, kv_heads;
  float scale_log2;  // |scale| log2(e), at least 1e-30 so that -inf stays -inf
  int negate;        // scale < 0: the queries' signs are flipped
  int causal;
  int64_t num_pages;
  int64_t q_stride;
  int warps_per_tile;  // 1, 2 or 4
  float* ws_o;         // [splits][tokens * heads][D]; splits > 1 only
  float2* ws_ml;       // [splits][tokens * heads]
  int32_t* status;
};

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  CTI_DEVICE static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static constexpr uint32_t kInf = 0x7f80u;
};
template <>
struct Mma<__half> {
  CTI_DEVICE static void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static constexpr uint32_t kInf = 0x7c00u;
};

CTI_DEVICE void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

template <typename T, int G, int ROWS>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(G))
    kv4_attention_kernel(const T* __restrict__ q, const uint8_t* __restrict__ pages, const Args a,
                         T* __restrict__ out) {
  using Y = Type16<T>;
  using M = Mma<T>;
  constexpr int D = 32 * G;
  constexpr int S = stages(G);
  constexpr int kBlock = block_bytes(G);
  constexpr bool kTwo = ROWS == 16;  // rows 8..15 are in use
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = warp_id(), lane = lane_id();
  const int r8 = lane >> 2, t4 = lane & 3;
  uint8_t* ring = smem + (size_t)warp * S * kBlock;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)kWarps * S * kBlock) + warp * S;
  if (lane == 0) {
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  grid_dependency_wait();

  const int wpt = a.warps_per_tile;
  const int64_t unit = (int64_t)blockIdx.x * (kWarps / wpt) + warp / wpt;
  if (unit >= (int64_t)a.num_seqs * a.kv_heads) return;  // all warps of a tile alike
  const int sub = warp & (wpt - 1);
  const int s = (int)(unit / a.kv_heads), kvh = (int)(unit % a.kv_heads);
  const int group = a.heads / a.kv_heads;
  int64_t begin = __ldg(a.cu + s), end = __ldg(a.cu + s + 1);
  const int64_t len = __ldg(a.kv_lens + s);
  const int64_t n_given = end - begin;
  const int64_t first = len - n_given;  // position of the first new token
  if (begin < 0 || end > a.tokens || n_given < 0) {
    if (lane == 0) raise_status(a.status, CTI_ERR_INVALID_ARG, s);
    return;
  }
  const int64_t rows = n_given * group;
  int64_t limit = len;  // keys that the table reaches
  if (limit > (int64_t)a.table_cols * kPage || (limit > 0 && a.num_pages <= 0)) {
    if (lane == 0 && rows > 0) raise_status(a.status, CTI_ERR_BOUNDS, s);
    limit = a.num_pages <= 0 ? 0 : (int64_t)a.table_cols * kPage;
  }
  const int32_t* table = a.table + s * a.table_stride;
  const uint8_t* base = pages + (int64_t)kvh * kBlock;
  const int64_t page_stride = (int64_t)a.kv_heads * kBlock;
  const float sl = a.scale_log2;
  uint32_t count = 0;  // pages copied so far: stage and parity
  bool dead = false;   // a copy did not arrive in time

  for (int64_t tile = blockIdx.y; tile * ROWS < rows; tile += gridDim.y) {
    // ---- rows: queries, keys that each sees ----
    int64_t row_at[2];  // output row (token * heads + head), -1: none
    int64_t sees[2];    // keys
    uint32_t qa[G][2][4];
    uint32_t off_a[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t r = tile * ROWS + r8 + 8 * e;
      const bool live = (e == 0 || kTwo) && r < rows;
      const int64_t i = live ? r / group : 0;
      const int h = kvh * group + (int)(r - i * group);
      row_at[e] = live ? (begin + i) * a.heads + h : -1;
      sees[e] = live ? (a.causal ? min(first + i + 1, limit) : limit) : 0;
      float sum_mine = 0.0f;  // of group t4's 32 dims (G = 2: t4 & 1; G = 1: the only one)
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live)
          v = __ldg(reinterpret_cast<const uint4*>(q + (begin + i) * a.q_stride + (int64_t)h * D +
                                                   32 * g + 8 * t4));
        if (a.negate) {
          v.x ^= 0x80008000u;
          v.y ^= 0x80008000u;
          v.z ^= 0x80008000u;
          v.w ^= 0x80008000u;
        }
        qa[g][0][e] = v.x;
        qa[g][0][2 + e] = v.y;
        qa[g][1][e] = v.z;
        qa[g][1][2 + e] = v.w;
        float sum = Y::low(v.x) + Y::high(v.x) + Y::low(v.y) + Y::high(v.y) + Y::low(v.z) +
                    Y::high(v.z) + Y::low(v.w) + Y::high(v.w);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (g == (t4 & (G - 1))) sum_mine = sum;
      }
      // The bases' operand: column 2 t + 1 multiplies b of the group that the
      // matching word of K's meta holds; column 2 t (its scale) gets 0.
      const uint32_t hi = Y::bits(sum_mine);
      const uint32_t lo = Y::bits(sum_mine - Y::to_float(hi));
      if (G == 4) {
        off_a[e] = hi << 16;
        off_a[2 + e] = lo << 16;
      } else {
        off_a[e] = t4 < G ? hi << 16 : t4 < 2 * G ? lo << 16 : 0u;
      }
    }
    // Keys that some row and that every row of the tile sees.
    const int64_t r_last = min(rows, (tile + 1) * ROWS) - 1;
    const int64_t most =
        max(a.causal ? min(first + r_last / group + 1, limit) : limit, (int64_t)0);
    const int64_t all = a.causal ? min(first + tile * ROWS / group + 1, limit) : limit;

    float o[4 * G][4];
#pragma unroll
    for (int i = 0; i < 4 * G; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    // ---- this warp's pages ----
    const int64_t npages = (most + kPage - 1) / kPage;
    const int workers = gridDim.z * wpt;
    const int64_t per = (npages + workers - 1) / workers;
    const int64_t p0 = min(npages, per * (blockIdx.z * wpt + sub));
    const int np = dead ? 0 : (int)(min(npages, p0 + per) - p0);
    int ids = -1;  // lane i: page p0 + (chunk of 32) + i
    auto load_ids = [&](int i) {
      ids = i + lane < np ? __ldg(table + p0 + i + lane) : 0;
      if (ids < 0 || ids >= a.num_pages) {
        raise_status(a.status, CTI_ERR_BOUNDS, s);
        ids = -1;
      }
    };
    uint32_t bad = 0;  // bit per page in flight (by stage): not a page, nothing of it is seen
    auto issue = [&](int i) {  // page i of the range into its stage
      if ((i & 31) == 0) load_ids(i);
      int id = __shfl_sync(0xffffffffu, ids, i & 31);
      const uint32_t st = (count + i) % S;
      bad = id < 0 ? bad | 1u << st : bad & ~(1u << st);
      if (id < 0) id = 0;
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[st], kBlock);
        bulk_load(ring + st * kBlock, base + id * page_stride, kBlock, &full[st]);
      }
    };
    for (int i = 0; i < S && i < np; ++i) issue(i);

    int done = 0;
    for (; done < np; ++done) {
      const uint32_t st = (count + done) % S;
      if (!__all_sync(0xffffffffu, mbar_wait(&full[st], ((count + done) / S) & 1, a.status, 0x700,
                                             nullptr)))
        break;
      uint8_t* blk = ring + st * kBlock;
      const int64_t key0 = (p0 + done) * kPage;
      const bool is_bad = (bad >> st) & 1;
      const bool whole = !is_bad && key0 + kPage <= all;

      // ---- S = Q K^T ----
      float sc[8][4];
#pragma unroll
      for (int v = 0; v < 2 * G; ++v) {
        const uint4 w4 = *reinterpret_cast<const uint4*>(blk + (v * 32 + lane) * 16);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int nt = (4 * v + j) / G, g = (4 * v + j) % G;
          if (g == 0) {
            const uint32_t meta = *reinterpret_cast<const uint32_t*>(
                blk + k_meta_at(G) + ((8 * nt + r8) * G + (t4 & (G - 1))) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[nt][e] = 0.0f;
            M::run(sc[nt], off_a, meta, G == 4 ? meta : 0u);
          }
          float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          M::run(c, qa[g][0], k_pair<T>(w[j], 0), k_pair<T>(w[j], 1));
          M::run(c, qa[g][1], k_pair<T>(w[j], 2), k_pair<T>(w[j], 3));
          const uint32_t* mc = reinterpret_cast<const uint32_t*>(blk + k_meta_at(G)) +
                               (8 * nt + 2 * t4) * G + g;
          const float s0 = Y::low(mc[0]), s1 = Y::low(mc[G]);
          sc[nt][0] = fmaf(c[0], s0, sc[nt][0]);
          sc[nt][1] = fmaf(c[1], s1, sc[nt][1]);
          if (kTwo) {
            sc[nt][2] = fmaf(c[2], s0, sc[nt][2]);
            sc[nt][3] = fmaf(c[3], s1, sc[nt][3]);
          }
        }
      }

      if (!whole) {
        // Keys that a row does not see count nothing, whatever they hold.  A
        // value that is not finite must reach only the rows that see it: its
        // scores become NaN for them, and its meta zero for all.
        const int64_t lim0 = is_bad ? 0 : sees[0] - key0, lim1 = is_bad ? 0 : sees[1] - key0;
        const int64_t lim_most = is_bad ? 0 : most - key0;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) {
          const int tau = 8 * nt + 2 * t4;
          uint32_t* vm = reinterpret_cast<uint32_t*>(blk + v_meta_at(G)) + (4 * nt + t4) * 2 * G;
          bool nan0 = false, nan1 = false;
#pragma unroll
          for (int i = 0; i < 2 * G; ++i) {
            nan0 |= (vm[i] & M::kInf) == M::kInf;
            nan1 |= ((vm[i] >> 16) & M::kInf) == M::kInf;
          }
          __syncwarp();
          if (nan0 || tau >= lim_most)
            for (int i = 0; i < 2 * G; ++i) vm[i] &= 0xffff0000u;
          if (nan1 || tau + 1 >= lim_most)
            for (int i = 0; i < 2 * G; ++i) vm[i] &= 0x0000ffffu;
          if (nan0) sc[nt][0] = sc[nt][2] = NAN;
          if (nan1) sc[nt][1] = sc[nt][3] = NAN;
          if (tau >= lim0) sc[nt][0] = -INFINITY;
          if (tau + 1 >= lim0) sc[nt][1] = -INFINITY;
          if (tau >= lim1) sc[nt][2] = -INFINITY;
          if (tau + 1 >= lim1) sc[nt][3] = -INFINITY;
        }
        fence_proxy_async_smem();
        __syncwarp();
      }

      // ---- the rows' exponent offsets ----
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        mx[0] = fmaxf(mx[0], fmaxf(sc[nt][0], sc[nt][1]));
        if (kTwo) mx[1] = fmaxf(mx[1], fmaxf(sc[nt][2], sc[nt][3]));
      }
      const bool raise = (mx[0] - m[0]) * sl > kSlack || (kTwo && (mx[1] - m[1]) * sl > kSlack);
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int e = 0; e < (kTwo ? 2 : 1); ++e) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
          if (mx[e] > m[e]) {
            const float corr = ex2_approx((m[e] - mx[e]) * sl);
            m[e] = mx[e];
            l[e] *= corr;
#pragma unroll
            for (int i = 0; i < 4 * G; ++i) {
              o[i][2 * e] *= corr;
              o[i][2 * e + 1] *= corr;
            }
          }
        }
      }
      const float off0 = m[0] == -INFINITY ? 0.0f : m[0] * sl;
      const float off1 = m[1] == -INFINITY ? 0.0f : m[1] * sl;

      // ---- P, and O += P V, 16 keys at a time ----
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t pa[4] = {0, 0, 0, 0};
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          float(&x)[4] = sc[2 * kk + hh];
          x[0] = ex2_approx(fmaf(x[0], sl, -off0));
          x[1] = ex2_approx(fmaf(x[1], sl, -off0));
          l[0] += x[0] + x[1];
          pa[2 * hh] = Y::pack(x[0], x[1]);
          if (kTwo) {
            x[2] = ex2_approx(fmaf(x[2], sl, -off1));
            x[3] = ex2_approx(fmaf(x[3], sl, -off1));
            l[1] += x[2] + x[3];
            pa[2 * hh + 1] = Y::pack(x[2], x[3]);
          }
        }
        const uint2* vm = reinterpret_cast<const uint2*>(blk + v_meta_at(G)) + (8 * kk + t4) * G;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint2 m0 = vm[g], m1 = vm[4 * G + g];
          const int i0 = 2 * kk * G + g, i1 = i0 + G;
          const uint32_t w0 = *reinterpret_cast<const uint32_t*>(
              blk + v_codes_at(G) + ((i0 >> 2) * 32 + lane) * 16 + (i0 & 3) * 4);
          const uint32_t w1 = *reinterpret_cast<const uint32_t*>(
              blk + v_codes_at(G) + ((i1 >> 2) * 32 + lane) * 16 + (i1 & 3) * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            M::run(o[4 * g + j], pa, fma2<T>(v_pair<T>(w0, j), m0.x, m0.y),
                   fma2<T>(v_pair<T>(w1, j), m1.x, m1.y));
        }
      }
      __syncwarp();
      if (done + S < np) issue(done + S);
    }
    if (done < np) {  // let the copies in flight land, then give up
      dead = true;
      for (int i = done; i < np && i < done + S; ++i)
        mbar_wait(&full[(count + i) % S], ((count + i) / S) & 1, a.status, 0x701, nullptr);
    }
    count += np;

    // ---- join and store ----
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
    if (wpt > 1) {
      // Every warp's rows in its own ring, then the first warp adds them up.
      const int bar = 1 + warp / wpt;
      float* mine = reinterpret_cast<float*>(ring);
      float* ml = mine + ROWS * D;
      static_assert((ROWS * D + 2 * ROWS) * 4 <= S * kBlock, "room for the rows");
      __syncwarp();
      if (sub != 0) {
#pragma unroll
        for (int e = 0; e < (kTwo ? 2 : 1); ++e) {
          float* dst = mine + (r8 + 8 * e) * D + 8 * t4;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float4* d4 = reinterpret_cast<float4*>(dst + 32 * g);
            d4[0] = make_float4(o[4 * g][2 * e], o[4 * g + 1][2 * e], o[4 * g + 2][2 * e],
                                o[4 * g + 3][2 * e]);
            d4[1] = make_float4(o[4 * g][2 * e + 1], o[4 * g + 1][2 * e + 1],
                                o[4 * g + 2][2 * e + 1], o[4 * g + 3][2 * e + 1]);
          }
          if (t4 == 0) {
            ml[2 * (r8 + 8 * e)] = m[e];
            ml[2 * (r8 + 8 * e) + 1] = l[e];
          }
        }
      }
      named_barrier_sync(bar, 32 * wpt);
      if (sub == 0) {
        for (int w = 1; w < wpt; ++w) {
          const float* src = reinterpret_cast<const float*>(ring + (size_t)w * S * kBlock);
          const float* src_ml = src + ROWS * D;
#pragma unroll
          for (int e = 0; e < (kTwo ? 2 : 1); ++e) {
            const float mw = src_ml[2 * (r8 + 8 * e)], lw = src_ml[2 * (r8 + 8 * e) + 1];
            const float mm = fmaxf(m[e], mw);
            const float ca = m[e] == mm ? 1.0f : ex2_approx((m[e] - mm) * sl);
            const float cb = mw == mm ? 1.0f : ex2_approx((mw - mm) * sl);
            m[e] = mm;
            l[e] = l[e] * ca + lw * cb;
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const float4* s4 =
                  reinterpret_cast<const float4*>(src + (r8 + 8 * e) * D + 32 * g + 8 * t4);
              const float4 x = s4[0], y = s4[1];
              o[4 * g][2 * e] = o[4 * g][2 * e] * ca + x.x * cb;
              o[4 * g + 1][2 * e] = o[4 * g + 1][2 * e] * ca + x.y * cb;
              o[4 * g + 2][2 * e] = o[4 * g + 2][2 * e] * ca + x.z * cb;
              o[4 * g + 3][2 * e] = o[4 * g + 3][2 * e] * ca + x.w * cb;
              o[4 * g][2 * e + 1] = o[4 * g][2 * e + 1] * ca + y.x * cb;
              o[4 * g + 1][2 * e + 1] = o[4 * g + 1][2 * e + 1] * ca + y.y * cb;
              o[4 * g + 2][2 * e + 1] = o[4 * g + 2][2 * e + 1] * ca + y.z * cb;
              o[4 * g + 3][2 * e + 1] = o[4 * g + 3][2 * e + 1] * ca + y.w * cb;
            }
          }
        }
      }
    }
    if (sub == 0) {
#pragma unroll
      for (int e = 0; e < (kTwo ? 2 : 1); ++e) {
        if (row_at[e] < 0) continue;
        if (gridDim.z == 1) {
          const float inv = l[e] == 0.0f ? 0.0f : 1.0f / l[e];
          uint4* dst = reinterpret_cast<uint4*>(out + row_at[e] * D + 8 * t4);
#pragma unroll
          for (int g = 0; g < G; ++g)
            dst[4 * g] = make_uint4(
                Y::pack(o[4 * g][2 * e] * inv, o[4 * g + 1][2 * e] * inv),
                Y::pack(o[4 * g + 2][2 * e] * inv, o[4 * g + 3][2 * e] * inv),
                Y::pack(o[4 * g][2 * e + 1] * inv, o[4 * g + 1][2 * e + 1] * inv),
                Y::pack(o[4 * g + 2][2 * e + 1] * inv, o[4 * g + 3][2 * e + 1] * inv));
        } else {
          const int64_t at = (int64_t)blockIdx.z * a.tokens * a.heads + row_at[e];
          float4* dst = reinterpret_cast<float4*>(a.ws_o + at * D + 8 * t4);
#pragma unroll
          for (int g = 0; g < G; ++g) {
            dst[8 * g] = make_float4(o[4 * g][2 * e], o[4 * g + 1][2 * e], o[4 * g + 2][2 * e],
                                     o[4 * g + 3][2 * e]);
            dst[8 * g + 1] = make_float4(o[4 * g][2 * e + 1], o[4 * g + 1][2 * e + 1],
                                         o[4 * g + 2][2 * e + 1], o[4 * g + 3][2 * e + 1]);
          }
          if (t4 == 0) a.ws_ml[at] = make_float2(m[e], l[e]);
        }
      }
    }
    if (wpt > 1) {
      // The rings are free again (copies may overwrite them) once the first
      // warp has read them.
      fence_proxy_async_smem();
      named_barrier_sync(1 + warp / wpt, 32 * wpt);
    }
  }
}

// Joins the splits of every row: one warp per row.
template <typename T, int G>
__global__ void __launch_bounds__(128)
    kv4_join_kernel(const Args a, int splits, T* __restrict__ out) {
  using Y = Type16<T>;
  constexpr int D = 32 * G;
  grid_dependency_wait();
  const int64_t rows = (int64_t)a.tokens * a.heads;
  const int64_t row = (int64_t)blockIdx.x * 4 + warp_id();
  const int lane = lane_id();
  if (row >= rows) return;
  const int64_t t = row / a.heads;
  if (t < __ldg(a.cu) || t >= __ldg(a.cu + a.num_seqs)) return;
  float mm = -INFINITY;
  for (int z = lane; z < splits; z += 32) mm = fmaxf(mm, a.ws_ml[z * rows + row].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, x));
  float l = 0.0f, o[G];
#pragma unroll
  for (int g = 0; g < G; ++g) o[g] = 0.0f;
#pragma unroll 4
  for (int z = 0; z < splits; ++z) {
    const float2 ml = a.ws_ml[z * rows + row];
    const float w = ml.x == mm ? 1.0f : ex2_approx((ml.x - mm) * a.scale_log2);
    l = fmaf(ml.y, w, l);
#pragma unroll
    for (int g = 0; g < G; ++g)
      o[g] = fmaf(a.ws_o[(z * rows + row) * D + 32 * g + lane], w, o[g]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int g = 0; g < G; ++g)
    reinterpret_cast<uint16_t*>(out)[row * D + 32 * g + lane] = (uint16_t)Y::bits(o[g] * inv);
}

// How a call is laid out over the GPU; a function of the sizes alone.
struct Plan {
  int rows;            // rows of a tile
  int warps_per_tile;  // that share a tile's pages in a block
  int splits;          // blocks that share them
  int64_t tiles;       // row tiles of a sequence
};

Plan plan(int num_seqs, int64_t tokens, int max_new, int64_t max_kv_len, int heads, int kv_heads,
          int head_dim) {
  const int G = head_dim / kGroup;
  const int64_t most = max_new < tokens ? max_new : tokens;
  const int64_t rows = (most > 0 ? most : 1) * (heads / kv_heads);
  Plan p;
  p.rows = rows <= 8 ? 8 : 16;
  p.tiles = (rows + p.rows - 1) / p.rows;
  const double units = (double)num_seqs * kv_heads * (double)p.tiles;
  const int64_t pages = (max_kv_len + kPage - 1) / kPage;
  // Warps that run at once; a tile is shared by as many as leave none idle.
  const int64_t room = (int64_t)kSMs * blocks_per_sm(G) * kWarps;
  int64_t share = (int64_t)(room / units);
  share = share < 1 ? 1 : share > pages ? (pages > 0 ? pages : 1) : share;
  p.warps_per_tile = share >= 4 ? 4 : share >= 2 ? 2 : 1;
  p.splits = (int)(share / p.warps_per_tile);
  if (p.splits > 256) p.splits = 256;
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
  const int per = kWarps / p.warps_per_tile;
  const int64_t x = (units + per - 1) / per;
  if (x > INT32_MAX) return CTI_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)x, (unsigned)(p.tiles < 65535 ? p.tiles : 65535), (unsigned)p.splits);
  if (launch_dependent(kv4_attention_kernel<T, G, ROWS>, grid, dim3(kThreads), smem_bytes(G), s,
                       static_cast<const T*>(q), static_cast<const uint8_t*>(pages), a,
                       static_cast<T*>(out)) != cudaSuccess)
    return CTI_ERR_CUDA;
  if (p.splits > 1) {
    const int64_t blocks = ((int64_t)a.tokens * a.heads + 3) / 4;
    if (blocks > INT32_MAX) return CTI_ERR_UNSUPPORTED;
    if (launch_dependent(kv4_join_kernel<T, G>, dim3((unsigned)blocks), dim3(128), 0, s, a,
                         p.splits, static_cast<T*>(out)) != cudaSuccess)
      return CTI_ERR_CUDA;
  }
  return CTI_OK;
}

template <typename T, int G>
int launch_rows(const void* q, const void* pages, const Args& a, const Plan& p, void* out,
                cudaStream_t s) {
  return p.rows == 8 ? launch<T, G, 8>(q, pages, a, p, out, s)
                     : launch<T, G, 16>(q, pages, a, p, out, s);
}

template <typename T>
int launch_dim(const void* q, const void* pages, const Args& a, const Plan& p, int head_dim,
               void* out, cudaStream_t s) {
  return head_dim == 32   ? launch_rows<T, 1>(q, pages, a, p, out, s)
         : head_dim == 64 ? launch_rows<T, 2>(q, pages, a, p, out, s)
                          : launch_rows<T, 4>(q, pages, a, p, out, s);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

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
  if (tokens > INT32_MAX - 256 || heads > 65535) return CTI_ERR_UNSUPPORTED;
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
  const Args a = {cu_seqlens,
                  kv_lens,
                  page_table,
                  table_stride,
                  table_cols,
                  num_seqs,
                  (int)tokens,
                  heads,
                  kv_heads,
                  fmaxf(fabsf(scale) * kLog2e, 1e-30f),
                  scale < 0.0f,
                  causal,
                  num_pages,
                  q_stride,
                  p.warps_per_tile,
                  static_cast<float*>(workspace),
                  reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + ws_o),
                  status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == CTI_DTYPE_BF16 ? launch_dim<__nv_bfloat16>(q, pages, a, p, head_dim, out, s)
                                 : launch_dim<__half>(q, pages, a, p, head_dim, out, s);
}
