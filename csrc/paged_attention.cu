// Attention of one new token per sequence over a key / value cache in pages.
//
//   o[r, h] = sum_j softmax_j(scale * q[r, h] . k_j) v_j,   j < lens[r],
//
// where key j of row r is token j % page of page table[r, j / page], and the query heads h of a group share kv head h / G.  A row of
// length zero gives zeros.  Positions from lens[r] on are never read as numbers: what lies there may be anything.  A page number
// outside the pool hides its keys and records kBadPage in the status word, which the host turns into an exception.
//
// paged_attention_kernel reads every key and value once for all heads of its group (once for 16 in bf16, 8 above 128 features; 8 in fp32, 4 above
// 128).  The keys of all (row, kv head) pairs, "jobs", are one
// sequence of rounds, 8 KB of keys and values or a little more, that is dealt out evenly: a CTA an SM takes a contiguous range, each of its
// warps a contiguous part of that, so lengths from one token to the longest mix without an idle SM and without the host knowing them.
// A warp keeps the running maximum, sum and weighted values of its job in registers.  Parts of a job that fell to several warps are joined in
// shared memory, and of several CTAs through a workspace by the last of them to finish (a counter, no waiting; parts are added in order, so
// results repeat to the bit).
//
// Loads: TMA tiles of 128-byte rows, 128-byte swizzled, a ring of rounds for every warp that runs on across jobs; a few instructions a round
// for any strides and page sizes (a page that a round does not fit into is fetched in several boxes).  The features of a fragment are dealt to
// the lanes in another order than the matrix instruction's, and the keys of a round too, in all its operands alike, which a sum does not
// notice: so a lane reads 16 bytes at a time, and the eight lanes of a read fall on different banks.  Head sizes, strides and addresses off 16 bytes
// have the same rounds filled element by element, by the warp that works on them.
//
// bf16: S^T = K Q^T and O^T = V^T P^T by mma.sync, the group's heads as the 8 columns (two tiles of them for 9 to 16 heads); the bound is
// the cache stream, and a tcgen05 tile of 128 rows would be padding for the most part.  The weights enter as three bf16 parts, all 24 bits of
// them, and what a round's products add up to goes into the running values in fp32, rounded to nearest.  With two parts and values that ran on in the
// instructions' own accumulators, which truncate, one output in 450 of 32 sequences of 1 to 4096 keys and one in 240 of four of 65000 to 131072 was a step
// off its rounding; one in 3000 and 4000 is.  What that costs: nothing on the 32 sequences; 16 sequences of 4096 keys, 8 heads of 64, take 31.1 us
// instead of 30.2, 16 of 2048, 8 heads of 256 on 4, 33.4 instead of 31.7; the four take 247 us instead of 244, and for seconds on end, at the power limit,
// 270 instead of 256.
// fp32: multiply-adds, 8 lanes a key; they bound groups of four heads and more.
//
// Device time on B200, pages of 16 tokens in random order, middle values of several runs on several GPUs: bf16, 32 heads of 128 on 8: four sequences of
// 65000 to 131072 keys 247 us (243 to 253; 6.5 TB/s, the rate of a plain copy), 32 sequences of 1 to 4096 53.8 us (5.0 TB/s; its floor is 41), 32 of 2048
// 52 us, one of 2048 15 us.  One sequence of 65 keys, 12 heads of 64: 6.8 us.  fp32, 13 sequences of up to 1531 keys, 10 heads of 80 on 5: 18.5 us; 32 of
// 2048, 32 heads of 128 on 8: 104 us.  Filled element by element the 32 sequences of 2048 keys take 180 us in bf16 and 185 us in fp32, the one of 65 keys
// 10.5 us.
#include <cuda_bf16.h>

#include "common/host.h"
#include "common/ptx.cuh"
#include "common/reduce.cuh"

namespace dptb {

struct PagedAttnArgs {
  const void* q;       // [rows, heads, hd]
  const void* k;       // [pages, kv_heads, page, hd]
  const void* v;
  void* o;             // [rows, heads, hd]
  const int* table;    // [rows, width]
  const int* lens;     // [rows]
  long long q_row, q_head, o_row, o_head;                  // strides in elements; features are contiguous
  long long k_page, k_head, k_tok, v_page, v_head, v_tok;
  long long table_row;
  int rows, heads, kv_heads, hd, page, width, pages, f32;
  float scale;
  float* ws;           // parts of jobs that several CTAs share
  long long ws_floats;
  unsigned* counters;  // zeroed words, one per CTA; zero again afterwards
  int num_counters;
  // pos / page = pos * page_mul >> page_shift for 0 <= pos < 2^31 (set by the launcher): page_mul = ceil(2^page_shift / page) with
  // 2^(page_shift - 31) >= page, so the excess of page_mul adds less than 2^31 * page / 2^page_shift <= 1 quotient's last place.
  unsigned page_mul, page_shift;
};
static_assert(sizeof(PagedAttnArgs) == 216, "packed by the caller");

__device__ __forceinline__ int slot_of(const PagedAttnArgs& a, int pos) { return (int)((unsigned long long)pos * a.page_mul >> a.page_shift); }

// ------------------------------------------------------------------------------------------------------------ pieces
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// `bytes`, a multiple of 16, between 16-byte boundaries; they count on `bar`.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint4 read_piece(uint32_t addr) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(addr) : "memory");
  return u;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// What of a round a lane looks up: the page of a position, from a window of 32 table entries that the lanes hold.  The first window of the
// row after is loaded a row ahead, so that rows of a few rounds do not wait for their table.
struct PageWindow {
  int row = -1, first = 0, entry = -1, next_row = -1, next_entry = -1;
  __device__ __forceinline__ int load(const PagedAttnArgs& a, int r, int slot, int len, int lane) const {
    return slot + lane <= slot_of(a, len - 1) ? a.table[r * a.table_row + slot + lane] : -1;
  }
  __device__ __forceinline__ void cover(const PagedAttnArgs& a, int r, int slot, int last, int len, int lane) {
    if (r != row || slot < first || last >= first + 32) {
      entry = r == next_row && slot == 0 ? next_entry : load(a, r, slot, len, lane);
      row = r;
      first = slot;
    }
  }
  __device__ __forceinline__ void ahead(const PagedAttnArgs& a, int r, int len, int lane) {
    next_row = r;
    next_entry = load(a, r, 0, len, lane);
  }
  // (every lane of the warp calls it)
  __device__ __forceinline__ int at(int slot) const { return __shfl_sync(0xffffffffu, entry, (slot - first) & 31); }
};

// A place in the sequence of rounds: round k of the n rounds of job (row, vh); vh counts kv heads and within them tiles of query heads.
struct Cursor {
  int row, vh, k, n, kv;
  int unit;      // its number in the sequence
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTiny = 1.2e-38f;
constexpr float kNoHead = 1.0e30f;      // maximum of a column without a head: its weights are zero, and products of zeros take little power
constexpr int kMaxHeadDim = 256;
constexpr int kAlone = 2, kSnap = 3;      // rounds of a warp that may be had for no joins across CTAs

// ------------------------------------------------------------------------------------------------------------ bf16
// HD: features of a head, padded with zeros; NT: tiles of 8 query heads; M: times 16 keys a round (two for heads of up to 64 features: a
// request and a maximum for each 16 keys kept 16 sequences of 4096 at 39 us, each 32 take 32 us).
template <int HD, int NT, int M>
struct Bf16Round {
  using T = __nv_bfloat16;
  static constexpr int kKeys = 16 * M, kKeyShift = M == 2 ? 5 : 4, kHeads = 8 * NT, kHD = HD;
  static constexpr int kSegs = HD / 64, kSeg = kKeys * 128, kBytes = 2 * kSegs * kSeg;   // keys, then values: a tile for every 64 features
  static constexpr int kQueryBytes = kHeads * HD * 2;

  uint4 q[NT][HD / 32];       // head lane / 4, pieces (lane % 4) + 4 i
  float m[NT][2], l[NT][2];   // heads (lane % 4) * 2 and the next; l: of this lane's keys
  float o[NT][HD / 64][4][4]; // features 8 (order(lane / 4) + 8 b) + 2 i and the next, of those heads

  // Which key of a half round is row i of a fragment, and which piece of 8 features a lane takes: neighbours in a read differ in bit 2.
  static __device__ __forceinline__ int order(int i) { return i >> 1 | (i & 1) << 2; }

  // `queries`: those of the job, [kHeads][HD]; beyond `count` heads and a.hd features it holds anything.
  __device__ __forceinline__ void start(const PagedAttnArgs& a, const unsigned char* queries, int count, int lane) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = n * 8 + (lane >> 2);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const int f = ((lane & 3) + 4 * i) * 8;
        q[n][i] = h < count && f < a.hd ? *reinterpret_cast<const uint4*>(queries + (h * HD + f) * 2) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = n * 8 + (lane & 3) * 2 + e < count ? -INFINITY : kNoHead;
        l[n][e] = 0.0f;
      }
#pragma unroll
      for (int b = 0; b < HD / 64; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][b][i][e] = 0.0f;
    }
  }

  // `keys`: bit j, whether key j of the round is one.
  __device__ __forceinline__ void compute(uint32_t ring, unsigned keys, float scale2, const unsigned char*, int lane) {
    const int t = lane & 3, mine = order(lane >> 2);
    const uint32_t swz = (mine ^ t) << 4;              // piece t of row `mine`, and piece `mine` of row t
    const uint32_t kr = ring + mine * 128, vr = ring + kSegs * kSeg + t * 128;
    float sc[NT][M][2][4] = {};
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int b = 0; b < M; ++b) {
        const uint32_t at = kr + (i >> 1) * kSeg + b * 2048 + (swz ^ (i & 1) << 6);
        const uint4 k0 = read_piece(at), k1 = read_piece(at + 1024);
        const uint32_t fa[4] = {k0.x, k1.x, k0.y, k1.y}, fb[4] = {k0.z, k1.z, k0.w, k1.w};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_bf16_16816(sc[n][b][0], fa, q[n][i].x, q[n][i].y);
          mma_bf16_16816(sc[n][b][1], fb, q[n][i].z, q[n][i].w);
        }
      }
    const unsigned there = keys >> mine;               // bits 0, 8, ...: this lane's keys
    float corr[NT][2];
    uint32_t pp[NT][M][3][2];   // [16 keys][part][keys, keys + 8]: pairs of keys of head lane / 4
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float p[2 * M][2];   // [key, key + 8, ...][head]
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float s[2 * M], mx = -INFINITY;
#pragma unroll
        for (int r = 0; r < 2 * M; ++r) {
          const float x = (sc[n][r >> 1][0][2 * (r & 1) + e] + sc[n][r >> 1][1][2 * (r & 1) + e]) * scale2;
          s[r] = there >> (8 * r) & 1 ? x : -INFINITY;
          mx = fmaxf(mx, s[r]);
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float nm = fmaxf(m[n][e], mx), sub = nm == -INFINITY ? 0.0f : nm;
        corr[n][e] = exp2_fast(m[n][e] - sub);
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 2 * M; ++r) {
          p[r][e] = there >> (8 * r) & 1 ? exp2_fast(s[r] - sub) : 0.0f;
          sum += p[r][e];
        }
        l[n][e] = l[n][e] * corr[n][e] + sum;
        m[n][e] = nm;
      }
      // All 24 bits of a weight: its leading 8, the next, the rest.  Parts of a positive weight stay positive: its product with an infinite value is
      // infinite in each.
#pragma unroll
      for (int r = 0; r < 2 * M; ++r) {
        float rest[2] = {p[r][0], p[r][1]};
        const float tiny[2] = {fminf(p[r][0], kTiny), fminf(p[r][1], kTiny)};
#pragma unroll
        for (int part = 0; part < 3; ++part) {
          const uint32_t u0 = __float_as_uint(rest[0]), u1 = __float_as_uint(rest[1]);
          pp[n][r >> 1][part][r & 1] = movmatrix_trans((u0 >> 16) | (u1 & 0xffff0000u));
          rest[0] = fmaxf(rest[0] - __uint_as_float(u0 & 0xffff0000u), tiny[0]);
          rest[1] = fmaxf(rest[1] - __uint_as_float(u1 & 0xffff0000u), tiny[1]);
        }
      }
    }
    // A round's products are summed on their own and added to the running values by multiply-adds: the matrix instructions cut
    // off what does not fit their sums, so values that ran on in them would shrink by up to 2^-24 a step (8e-6 of them after 512 rounds).
#pragma unroll
    for (int b = 0; b < HD / 64; ++b) {
      uint32_t v[M][4][4];
#pragma unroll
      for (int c = 0; c < M; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 u = read_piece(vr + b * kSeg + c * 2048 + j * 512 + (swz ^ (j & 1) << 6));       // keys t, t + 4, t + 8, t + 12
          v[c][j][0] = u.x; v[c][j][1] = u.y; v[c][j][2] = u.z; v[c][j][3] = u.w;
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float sum[NT][4] = {};
#pragma unroll
        for (int c = 0; c < M; ++c) {
          const uint32_t f[4] = {__byte_perm(v[c][0][i], v[c][1][i], 0x5410), __byte_perm(v[c][0][i], v[c][1][i], 0x7632),
                                 __byte_perm(v[c][2][i], v[c][3][i], 0x5410), __byte_perm(v[c][2][i], v[c][3][i], 0x7632)};
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int part = 0; part < 3; ++part) mma_bf16_16816(sum[n], f, pp[n][c][part][0], pp[n][c][part][1]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][b][i][e] = fmaf(o[n][b][i][e], corr[n][e & 1], sum[n][e]);
      }
    }
  }

  __device__ __forceinline__ void finish(int lane) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], off);
  }
  // Eight consecutive features at a time: put(head, first feature, values, maximum, sum).
  template <typename F>
  __device__ __forceinline__ void each(int lane, F put) const {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int b = 0; b < HD / 64; ++b) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f[2 * i] = o[n][b][i][e];
            f[2 * i + 1] = o[n][b][i][2 + e];
          }
          put(n * 8 + (lane & 3) * 2 + e, 8 * (order(lane >> 2) + 8 * b), f, m[n][e], l[n][e]);
        }
  }
};

// ------------------------------------------------------------------------------------------------------------ fp32
// GP: query heads at a time.  Lane t of the 8 lanes of a key holds pieces t + 8 i of it; four keys go by at once, NJ steps a round.  The
// queries are read from shared memory where they are needed (features beyond the head's are zeros there).
//
// A round's products leave NJ GP sums of 8 lanes each (head, step).  They are added in halves: with every exchange a lane keeps half of its sums, so that
// in the end it has one or a few of one head, for which it alone keeps maximum and sum and takes the exponentials; the weights go
// back to the lanes by shuffle.  Multiply-adds are packed in pairs.  With every sum in every lane, and single multiply-adds, 13 sequences of up to
// 1531 keys (10 heads of 80 on 5) took 22 us, 18 so.  Rounds of 16 keys for heads of up to 64 features (16 sequences of 4096 keys: 65 us with 8, 51 with
// 16), of 8 above.
template <int HD, int GP, int NJ>
struct F32Round {
  using T = float;
  static constexpr int kKeys = 4 * NJ, kKeyShift = NJ == 4 ? 4 : 3, kHeads = GP, kHD = HD;
  static constexpr int P = HD / 32;                      // pieces of a key per lane
  static constexpr int kSegs = P, kSeg = kKeys * 128, kBytes = 2 * kSegs * kSeg;         // a tile for every 32 features
  static constexpr int kQueryBytes = GP * HD * 4;
  static constexpr int kSums = NJ * GP, kOwn = kSums > 8 ? kSums / 8 : 1, kSpread = kSums >= 8 ? 1 : 8 / kSums;     // sums; of a lane; lanes of a sum

  float m, l;
  f32x2 o[GP][P][2];

  // The lane (of 8) that keeps sum (head, step).
  static __device__ __forceinline__ constexpr int lane_of(int h, int j) { return (NJ * h + j) / kOwn * kSpread; }

  __device__ __forceinline__ void start(const PagedAttnArgs&, const unsigned char*, int, int) {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int h = 0; h < GP; ++h)
#pragma unroll
      for (int i = 0; i < P; ++i) o[h][i][0] = o[h][i][1] = 0ull;
  }

  __device__ __forceinline__ void compute(uint32_t ring, unsigned keys, float scale2, const unsigned char* queries, int lane) {
    const int g = lane >> 3, t = lane & 7;
    auto piece = [&](int seg, int j, f32x2 (&v)[2]) {    // of key g + 4 j
      const int key = g + 4 * j;
      const uint4 u = read_piece(ring + seg * kSeg + key * 128 + ((t ^ key & 7) << 4));
      v[0] = f2_pack(__uint_as_float(u.x), __uint_as_float(u.y));
      v[1] = f2_pack(__uint_as_float(u.z), __uint_as_float(u.w));
    };
    const ulonglong2* q = reinterpret_cast<const ulonglong2*>(queries) + t;
    float v[kSums];
    {
      f32x2 k[NJ][P][2];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < P; ++i) piece(i, j, k[j][i]);
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        f32x2 s[NJ] = {};
#pragma unroll
        for (int i = 0; i < P; ++i) {
          const ulonglong2 w = q[h * (HD / 4) + 8 * i];
#pragma unroll
          for (int j = 0; j < NJ; ++j) s[j] = f2_fma(k[j][i][1], w.y, f2_fma(k[j][i][0], w.x, s[j]));
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          float lo, hi;
          f2_unpack(s[j], lo, hi);
          v[NJ * h + j] = lo + hi;
        }
      }
    }
    int n = kSums;
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) {
      const bool upper = t & off;
      if (n > 1) {
        n >>= 1;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        }
      } else {
        v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
      }
    }
    float p[kOwn], mx = -INFINITY;
    bool live[kOwn];
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      const int j = (t / kSpread * kOwn + r) % NJ;
      live[r] = keys >> (g + 4 * j) & 1;
      p[r] = live[r] ? v[r] * scale2 : -INFINITY;
      mx = fmaxf(mx, p[r]);
    }
#pragma unroll
    for (int off = kSpread; off < 8 / GP; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));      // the head's other steps
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
    const float nm = fmaxf(m, mx), sub = nm == -INFINITY ? 0.0f : nm, corr = exp2_fast(m - sub);
    const bool moved = nm != m;
    l *= corr;
#pragma unroll
    for (int r = 0; r < kOwn; ++r) {
      p[r] = live[r] ? exp2_fast(p[r] - sub) : 0.0f;
      l += p[r];
    }
    m = nm;
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const f32x2 c = f2_splat(__shfl_sync(0xffffffffu, corr, lane & 24 | lane_of(h, 0)));
#pragma unroll
        for (int i = 0; i < P; ++i) {
          o[h][i][0] = f2_mul(o[h][i][0], c);
          o[h][i][1] = f2_mul(o[h][i][1], c);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      f32x2 w[GP];
#pragma unroll
      for (int h = 0; h < GP; ++h) w[h] = f2_splat(__shfl_sync(0xffffffffu, p[(NJ * h + j) % kOwn], lane & 24 | lane_of(h, j)));
#pragma unroll
      for (int i = 0; i < P; ++i) {
        f32x2 x[2];
        piece(kSegs + i, j, x);
#pragma unroll
        for (int h = 0; h < GP; ++h) {
          o[h][i][0] = f2_fma(w[h], x[0], o[h][i][0]);
          o[h][i][1] = f2_fma(w[h], x[1], o[h][i][1]);
        }
      }
    }
  }

  __device__ __forceinline__ void finish(int) {
#pragma unroll
    for (int off = kSpread; off < 8 / GP; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
#pragma unroll
    for (int off = 8; off < 32; off <<= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, off);
#pragma unroll
      for (int h = 0; h < GP; ++h)
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) o[h][i][e] = f2_add(o[h][i][e], __shfl_xor_sync(0xffffffffu, o[h][i][e], off));
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(int lane, F put) const {
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      const float mh = __shfl_sync(0xffffffffu, m, lane_of(h, 0)), lh = __shfl_sync(0xffffffffu, l, lane_of(h, 0));
      if (lane < 8)
#pragma unroll
        for (int i = 0; i < P; ++i) {
          float f[4];
          f2_unpack(o[h][i][0], f[0], f[1]);
          f2_unpack(o[h][i][1], f[2], f[3]);
          put(h, 4 * (lane + 8 * i), f, mh, lh);
        }
    }
  }
};

// ------------------------------------------------------------------------------------------------------------ the kernel
// A part of a job in memory: [heads][HD] weighted values, then the heads' maxima and sums.
template <typename R>
struct Part {
  static constexpr int kFloats = (R::kHeads * (R::kHD + 2) + 3) / 4 * 4;
};

struct PageMaps {
  CUtensorMap k, v;      // (feature, token of the page, head, page)
};

// All keys of a round, a bit each.
template <typename R>
__device__ __forceinline__ unsigned all_keys() { return R::kKeys == 32 ? 0xffffffffu : (1u << (R::kKeys & 31)) - 1; }

// A round that is not full, or of very small pages: in boxes of as many tokens as fit a page.  Out of line: the kernel's code is fetched anew at every
// launch, and most rounds do not come here.
template <typename R>
__device__ __noinline__ unsigned issue_boxes(const PagedAttnArgs& a, const PageMaps& maps, int entry, int first_slot, int kv, int p0, int len, int box_shift,
                                             unsigned char* ring, uint64_t* bar, int lane) {
  const int end = min(p0 + R::kKeys, len);
  auto page_of = [&](int slot) { return __shfl_sync(0xffffffffu, entry, slot - first_slot & 31); };
  if (lane == 0) mbar_arrive_expect_tx(bar, R::kBytes);
  const int pos = p0 + (lane & (R::kKeys - 1));
  const unsigned mine = page_of(slot_of(a, pos));
  const bool bad = pos < end && mine >= (unsigned)a.pages;
  if (bad) report_error(kBadPage);
  const unsigned keys = __ballot_sync(0xffffffffu, pos < end && !bad) & all_keys<R>();      // (orders the lanes before the copies too)
  const int per_shift = R::kKeyShift - box_shift, boxes = 2 * R::kSegs << per_shift;
#pragma unroll 1
  for (int b0 = 0; b0 < boxes; b0 += 32) {
    const int b = b0 + lane, first = (b & ((1 << per_shift) - 1)) << box_shift, tile = b >> per_shift;
    const int slot = slot_of(a, p0 + first);
    int page = page_of(slot);
    if ((unsigned)page >= (unsigned)a.pages) page = a.pages;                                            // beyond the pool: zeros
    if (b < boxes) {
      const bool is_v = tile >= R::kSegs;
      tma_load_4d(ring + tile * R::kSeg + first * 128, is_v ? &maps.v : &maps.k, bar, (is_v ? tile - R::kSegs : tile) * (128 / (int)sizeof(typename R::T)),
                  p0 + first - slot * a.page, kv, page);
    }
  }
  return keys;
}

// Requests the keys and values of round c; returns which of its keys there are.
template <typename R>
__device__ __forceinline__ unsigned issue_round(const PagedAttnArgs& a, const PageMaps& maps, PageWindow& win, const Cursor& c, int len, int box_shift,
                                                unsigned char* ring, uint64_t* bar, int lane) {
  const int p0 = c.k * R::kKeys, slot0 = slot_of(a, p0), per_shift = R::kKeyShift - box_shift, boxes = 2 * R::kSegs << per_shift;
  win.cover(a, c.row, slot0, slot_of(a, min(p0 + R::kKeys, len) - 1), len, lane);
  const int first = (lane & ((1 << per_shift) - 1)) << box_shift, tile = lane >> per_shift, slot = slot_of(a, p0 + first), page = win.at(slot);
  if (boxes > 32 || p0 + R::kKeys > len || __any_sync(0xffffffffu, lane < boxes && (unsigned)page >= (unsigned)a.pages))
    return issue_boxes<R>(a, maps, win.entry, win.first, c.kv, p0, len, box_shift, ring, bar, lane);
  if (lane == 0) mbar_arrive_expect_tx(bar, R::kBytes);
  __syncwarp();
  if (lane < boxes) {                              // a full round: a box a lane
    const bool is_v = tile >= R::kSegs;
    tma_load_4d(ring + tile * R::kSeg + first * 128, is_v ? &maps.v : &maps.k, bar, (is_v ? tile - R::kSegs : tile) * (128 / (int)sizeof(typename R::T)),
                p0 + first - slot * a.page, c.kv, page);
  }
  return all_keys<R>();
}

// The same for pages that TMA cannot fetch, element by element: by the warp itself, so that nothing is in flight afterwards.
template <typename R>
__device__ __forceinline__ unsigned fill_round(const PagedAttnArgs& a, PageWindow& win, const Cursor& c, int len, unsigned char* ring, int lane) {
  using T = typename R::T;
  const int p0 = c.k * R::kKeys, end = min(p0 + R::kKeys, len), slot0 = slot_of(a, p0);
  win.cover(a, c.row, slot0, slot_of(a, end - 1), len, lane);
  const int pos = p0 + (lane & (R::kKeys - 1)), slot = slot_of(a, pos), page = win.at(slot), tok = pos - slot * a.page;
  const bool bad = pos < end && (unsigned)page >= (unsigned)a.pages;
  if (bad) report_error(kBadPage);
  const unsigned keys = __ballot_sync(0xffffffffu, pos < end && !bad) & all_keys<R>();
  constexpr int kEach = R::kHD / 32, kAtOnce = 32 / kEach;      // elements of a lane; keys at a time
#pragma unroll 1
  for (int is_v = 0; is_v < 2; ++is_v) {
    const T* base = static_cast<const T*>(is_v ? a.v : a.k) + c.kv * (is_v ? a.v_head : a.k_head);
    const long long at = (long long)page * (is_v ? a.v_page : a.k_page) + (long long)tok * (is_v ? a.v_tok : a.k_tok);
    unsigned char* tile = ring + is_v * R::kSegs * R::kSeg;
#pragma unroll 1
    for (int j0 = 0; j0 < R::kKeys; j0 += kAtOnce) {
      T e[kAtOnce][kEach];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {        // (a load that depends on nothing: what there is not reads a query)
        const long long to = __shfl_sync(0xffffffffu, at, j0 + j);
        const T* src = keys >> (j0 + j) & 1 ? base + to : static_cast<const T*>(a.q);
#pragma unroll
        for (int i = 0; i < kEach; ++i) e[j][i] = src[min(lane + 32 * i, a.hd - 1)];
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int byte = (lane + 32 * i) * (int)sizeof(T), row = j0 + j;      // 128-byte swizzle, as a tile arrives
          *reinterpret_cast<T*>(tile + (byte >> 7) * R::kSeg + row * 128 + ((byte & 127) ^ (row & 7) << 4)) =
              (keys >> row & 1) && lane + 32 * i < a.hd ? e[j][i] : from_f32<T>(0.0f);
        }
    }
  }
  __syncwarp();
  return keys;
}

// And the queries of a job.
template <typename R>
__device__ __noinline__ void fill_queries(const typename R::T* src, typename R::T* dst, int heads, int hd, long long q_head, int lane) {
  constexpr int U = 8;
#pragma unroll 1
  for (int i0 = lane; i0 < heads * R::kHD; i0 += 32 * U) {
    typename R::T e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 32 * u, h = i / R::kHD, f = i - h * R::kHD;
      if (h < heads && f < hd) e[u] = src[h * q_head + f];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 32 * u, h = i / R::kHD, f = i - h * R::kHD;
      if (h < heads && f < hd) dst[i] = e[u];
    }
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_out(T* dst, const float (&f)[N], float by, int valid, bool vec) {
  T e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = from_f32<T>(f[i] * by);
  static_assert(N * sizeof(T) == 16, "a piece");
  if (vec && valid >= N) {
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(e);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < valid) dst[i] = e[i];
  }
}

// Parts of a job are joined, first those of this CTA (stage 0): of a job that lies within it, to the output; of another's, to the workspace, place 0
// of the CTA for the job of its first round, 1 for one that begins later.  The last CTA that gets so far with a job joins what the
// workspace holds of it (stage 1), in the order of the CTAs.  Warps take turns at (job, head); lane j has part j.  One loop for both.
template <int W>
struct Parts {
  int job[2 * W], row[2 * W], head[2 * W], count[2 * W], begin[2 * W], rounds[2 * W];
  int shared[2], merges[2];      // jobs of several CTAs: one of their parts here, or -1; whether this CTA is the last
};

template <typename R, int W, int S>
__device__ __noinline__ void join_parts(const PagedAttnArgs& a, Parts<W>& sh, const unsigned char* rings, const float* leads, int begin, int end, int share) {
  using T = typename R::T;
  constexpr int kPart = Part<R>::kFloats;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kPer = R::kHD / 32;                            // features of a lane
  constexpr int kMax = R::kHeads * R::kHD, kSum = kMax + R::kHeads;
#pragma unroll 1
  for (int stage = 0; stage < 2; ++stage) {
    unsigned jobs, same = 0;                                   // the jobs at hand: one of their parts in this CTA each
    if (stage == 0) {
      const int job = lane < 2 * W ? sh.job[lane] : -1;
      same = __match_any_sync(0xffffffffu, job);
      jobs = __ballot_sync(0xffffffffu, job >= 0 && (same & ((1u << lane) - 1)) == 0);
    } else {
      __syncthreads();
      if (sh.shared[0] < 0 && sh.shared[1] < 0) return;
      if (tid < 2) {
        const int i = sh.shared[tid];
        int last = 0;
        if (i >= 0) {
          const int first = sh.begin[i] / share, n = (sh.begin[i] + sh.rounds[i] - 1) / share - first;
          unsigned before;      // releases what this CTA has written (the barrier above), acquires what those before it have (the one below)
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + first) : "memory");
          last = before == (unsigned)n;
          if (last) a.counters[first] = 0;
        }
        sh.merges[tid] = last;
      }
      __syncthreads();
      jobs = (sh.merges[0] ? 1u << sh.shared[0] : 0) | (sh.merges[1] ? 1u << sh.shared[1] : 0);
    }
    int unit = 0;
#pragma unroll 1
    for (; jobs; jobs &= jobs - 1) {
      const int i = __ffs(jobs) - 1, jb = sh.begin[i], stop = jb + sh.rounds[i], heads = sh.count[i];
      const bool whole = jb >= begin && stop <= end;
      const unsigned group_of = __shfl_sync(0xffffffffu, same, i);
      if (stage == 0 && !whole && tid == 0) sh.shared[jb > begin] = i;
      const int first = stage ? jb / share : 0, n = stage ? (stop - 1) / share - first + 1 : 32;
#pragma unroll 1
      for (int h = 0; h < heads; ++h, ++unit) {
        if (unit % W != warp) continue;
        float m = -INFINITY, l = 0.0f, f[kPer] = {};
#pragma unroll 1
        for (int j0 = 0; j0 < n; j0 += 32) {
          const int j = j0 + lane;
          const float* part = nullptr;
          if (stage == 0) {
            if (group_of >> lane & 1) part = lane & 1 ? reinterpret_cast<const float*>(rings + (lane >> 1) * S * R::kBytes) : leads + (lane >> 1) * kPart;
          } else if (j < n) {
            part = a.ws + ((first + j) * 2LL + (j == 0 && jb > first * share)) * kPart;
          }
          // The values of the first parts are on their way while the weights are worked out.
          const float mine = part ? *(const volatile float*)(part + kMax + h) : -INFINITY, of = part ? *(const volatile float*)(part + kSum + h) : 0.0f;
          unsigned parts = __ballot_sync(0xffffffffu, part != nullptr);
          constexpr int kEarly = 3;
          float early[kEarly][kPer];
          int who[kEarly];
#pragma unroll
          for (int y = 0; y < kEarly; ++y) {
            who[y] = parts ? __ffs(parts) - 1 : 0;
            const volatile float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(part), who[y])) + h * R::kHD + lane;
#pragma unroll
            for (int e = 0; e < kPer; ++e) early[y][e] = parts ? src[32 * e] : 0.0f;
            if (!parts) who[y] = -1;
            parts &= parts - 1;
          }
          const float nm = fmaxf(m, warp_max(mine)), sub = nm == -INFINITY ? 0.0f : nm, corr = exp2_fast(m - sub);
          const float w = part ? exp2_fast(mine - sub) : 0.0f;
          l = l * corr + warp_sum(w * of);
          m = nm;
#pragma unroll
          for (int e = 0; e < kPer; ++e) f[e] *= corr;
#pragma unroll
          for (int y = 0; y < kEarly; ++y) {
            const float wy = __shfl_sync(0xffffffffu, w, max(who[y], 0));
            if (who[y] >= 0)
#pragma unroll
              for (int e = 0; e < kPer; ++e) f[e] += wy * early[y][e];
          }
#pragma unroll 4
          for (; parts; parts &= parts - 1) {
            const int x = __ffs(parts) - 1;
            const volatile float* src = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(part), x)) + h * R::kHD + lane;
            const float wx = __shfl_sync(0xffffffffu, w, x);
#pragma unroll
            for (int e = 0; e < kPer; ++e) f[e] += wx * src[32 * e];
          }
        }
        if (stage || whole) {
          T* out = static_cast<T*>(a.o) + sh.row[i] * a.o_row + (long long)(sh.head[i] + h) * a.o_head;
          const float by = 1.0f / l;
#pragma unroll
          for (int e = 0; e < kPer; ++e)
            if (lane + 32 * e < a.hd) out[lane + 32 * e] = from_f32<T>(f[e] * by);
        } else {
          float* dst = a.ws + (blockIdx.x * 2LL + (jb > begin)) * kPart;
#pragma unroll
          for (int e = 0; e < kPer; ++e) dst[h * R::kHD + lane + 32 * e] = f[e];
          if (lane == 0) {
            dst[kMax + h] = m;
            dst[kSum + h] = l;
          }
        }
      }
    }
  }
}

// W warps, S rounds of a warp in flight or in use.
template <typename R, int W, int S, bool TMA>
__global__ void __launch_bounds__(W * 32, 1)
paged_attention_kernel(const __grid_constant__ PagedAttnArgs a, const __grid_constant__ PageMaps maps, int box_shift, int head_tiles, int tile_heads,
                       int q_vec, int o_vec) {
  using T = typename R::T;
  constexpr int kPart = Part<R>::kFloats;
  static_assert(S * R::kBytes >= kPart * 4, "a warp's ring holds its last part");
  extern __shared__ unsigned char smem[];
  unsigned char* rings = smem + (1024 - (smem_u32(smem) & 1023) & 1023);      // [W][S] rounds
  float* leads = reinterpret_cast<float*>(rings + W * S * R::kBytes);       // [W] parts
  unsigned char* queries = reinterpret_cast<unsigned char*>(leads + W * kPart);   // [W][S] jobs' queries
  int* before = reinterpret_cast<int*>(queries + W * S * R::kQueryBytes);   // [rows + 1]: units of a kv head ahead of a row
  unsigned char* tails = reinterpret_cast<unsigned char*>(before + a.rows + 1);   // [rows]: tokens of a row's last round
  __shared__ int scan[W], most[W];
  __shared__ Parts<W> sh;
  __shared__ uint64_t landed[W * S];
  __shared__ int aborted;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tiles = a.kv_heads * head_tiles;                                // jobs of a row
  const int room = (int)min((long long)a.width * a.page, 0x7fffff00LL);      // (the end of its last round is a position, too)
  const int group = a.heads / a.kv_heads;

  // Units ahead of every row: a job is its rounds and, before them, one unit for what it costs to begin and end it (2100 cycles where a round took
  // 2500; without it the warps of the shortest rows came last by a quarter).
  auto length = [&](int r) { return max(0, min(a.lens[r], room)); };
  bool alone, snap, single;    // a job a CTA; CTAs of whole jobs; jobs of a round each
  {
    const int each = (a.rows + W * 32 - 1) / (W * 32), r0 = min(a.rows, tid * each), r1 = min(a.rows, r0 + each);
    int mine = 0, longest = 0;
    for (int r = r0; r < r1; ++r) {
      const int n = a.lens[r], k = (max(0, min(n, room)) + R::kKeys - 1) / R::kKeys;
      if (n > room && blockIdx.x == 0) report_error(kBadPage);
      mine += k + (k > 0);
      longest = max(longest, k);
    }
    int s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) scan[warp] = s;
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) most[warp] = longest;
    __syncthreads();
    int sum = 0, top = 0;
    for (int w = 0; w < W; ++w) {
      sum += scan[w];
      top = max(top, most[w]);
    }
    const bool few = a.rows * tiles <= gridDim.x;
    snap = !few && top <= kSnap * W;
    single = top <= 1;
    alone = few && (top + W - 1) / W <= (int)(((unsigned)(sum * tiles) + W * gridDim.x - 1) / (W * gridDim.x)) + kAlone;
    int at = s - mine;
    for (int w = 0; w < warp; ++w) at += scan[w];
    for (int r = r0; r < r1; ++r) {
      const int n = length(r);
      before[r] = at;
      tails[r] = n - (n - 1) / R::kKeys * R::kKeys;
      at += (n + R::kKeys - 1) / R::kKeys + (n > 0);
    }
    if (tid == 0) before[a.rows] = sum;
    if (tid < 2 * W) sh.job[tid] = -1;
    if (tid < 2) sh.shared[tid] = -1;
    if (a.hd < R::kHD)
      for (int i = tid; i < W * S * R::kQueryBytes / 16; i += W * 32) reinterpret_cast<uint4*>(queries)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    if (tid < W * S) mbar_init(landed + tid, 1);
    if (tid == 0) aborted = 0;
    mbar_fence_init();
    __syncthreads();
  }
  const int total = before[a.rows] * tiles;                    // (below 2^31: the launcher sees to it)
  auto row_of = [&](int unit) {        // the last row with no more units ahead, which has some itself; a warp looks at 32 at a time
    int row = 0;
    for (int n = a.rows; n > 1;) {
      const int step = (n + 31) / 32, at = lane * step;
      const int skip = (__popc(__ballot_sync(0xffffffffu, at < n && before[min(row + at, a.rows)] * tiles <= unit)) - 1) * step;
      row += skip;
      n = min(step, n - skip);
    }
    return row;
  };
  // A CTA takes a unit for each of its warps at least: parts of one CTA are joined sooner than those of several.  So a CTA takes a job, if there are no more of
  // them than CTAs and the longest keeps its warps for at most two rounds more than a share would (32 heads of 128 on 8, 16 sequences of 250 keys:
  // 10.8 us, shared 14.3; of 2000 keys 29.8 and 32.9; with five rounds more, 4 sequences of 800 keys take 16.3 instead of 14).  If there are more jobs and
  // all are short, a CTA takes those that begin in its share (32 sequences of up to 250 keys: 14.3 and 17.1; 1024 of 250, 8 heads on 2: 55 and 61).
  int share = max(W, (int)((unsigned)(total + gridDim.x - 1) / gridDim.x));
  if (single) share += share & 1;                              // two units each: no job is cut
  int begin = (int)min((long long)total, (long long)share * blockIdx.x), end = min(total, begin + share);
  if (alone) {
    const int row = min((int)blockIdx.x / tiles, a.rows), units = row < a.rows ? before[row + 1] - before[row] : 0;
    begin = before[row] * tiles + ((int)blockIdx.x - row * tiles) * units;
    end = begin + units;
  } else if (snap && !single) {
    auto start_of_job = [&](int unit) {                        // at `unit` or after it
      if (unit >= total) return total;
      const int row = row_of(unit), units = before[row + 1] - before[row], first = before[row] * tiles;
      return first + (unit - first + units - 1) / units * units;
    };
    begin = start_of_job(begin);
    end = start_of_job(end);
  }
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {       // rows of no tokens
    if (before[r + 1] > before[r]) continue;
    for (int x = tid; x < a.heads * a.hd; x += W * 32) static_cast<T*>(a.o)[r * a.o_row + x / a.hd * a.o_head + x % a.hd] = from_f32<T>(0.0f);
  }
  if (begin >= end) return;

  const int quota = (end - begin + W - 1) / W, w0 = min(end, begin + quota * warp), w1 = min(end, w0 + quota);
  if (w0 < w1) {
    unsigned char* ring = rings + warp * S * R::kBytes;
    uint64_t* bars = landed + warp * S;
    unsigned char* my_queries = queries + warp * S * R::kQueryBytes;
    const int row = row_of(w0);
    const int n0 = before[row + 1] - before[row] - 1, rem = w0 - before[row] * tiles, vh0 = rem / (n0 + 1), u0 = rem - vh0 * (n0 + 1);
    Cursor c{row, vh0, max(u0 - 1, 0), n0, head_tiles == 1 ? vh0 : vh0 / head_tiles, w0 + (u0 == 0)}, ahead = c;
    auto advance = [&](Cursor& x) {
      ++x.unit;
      if (++x.k < x.n) return;
      ++x.unit;
      x.k = 0;
      ++x.vh;
      x.kv = head_tiles == 1 ? x.vh : x.vh / head_tiles;
      if (x.vh < tiles) return;
      x.vh = x.kv = 0;
      do {
        ++x.row;
      } while (x.row < a.rows && before[x.row + 1] == before[x.row]);
      if (x.row < a.rows) x.n = before[x.row + 1] - before[x.row] - 1;
    };
    PageWindow win;
    static_assert(S * R::kKeys <= 64, "a bit for each key of the ring");
    unsigned long long there = 0;
    int put = 0, take = 0, len = 0, len_row = -1, put_job = 0, take_job = 0;
    bool new_job = true;
    auto length_of = [&](int r) { return (before[r + 1] - before[r] - 2) * R::kKeys + tails[r]; };
    auto fetch = [&] {
      if (ahead.unit >= w1) return;
      if (ahead.row != len_row) {
        len_row = ahead.row;
        len = length_of(len_row);
      }
      uint64_t* bar = bars + put;
      if (new_job) {
        // The job's queries come with its first round: loaded when the job starts, they cost each job the latency of the memory.  A place is free
        // again when the job S before is done: a fetch is at most S - 1 rounds ahead.
        const int tile = ahead.vh - ahead.kv * head_tiles, heads = min(tile_heads, group - tile * tile_heads);
        const T* src = static_cast<const T*>(a.q) + ahead.row * a.q_row + (long long)(ahead.kv * group + tile * tile_heads) * a.q_head;
        T* dst = reinterpret_cast<T*>(my_queries + put_job * R::kQueryBytes);
        const int bytes = a.hd * (int)sizeof(T);
        if (TMA && q_vec) {
          if (lane == 0) mbar_expect_tx(bar, heads * bytes);
          __syncwarp();
          if (lane < heads) bulk_load(dst + lane * R::kHD, src + lane * a.q_head, bytes, bar);
        } else {
          fill_queries<R>(src, dst, heads, a.hd, a.q_head, lane);
        }
        __syncwarp();
        put_job = put_job + 1 == S ? 0 : put_job + 1;
      }
      unsigned keys;
      if constexpr (TMA) keys = issue_round<R>(a, maps, win, ahead, len, box_shift, ring + put * R::kBytes, bar, lane);
      else               keys = fill_round<R>(a, win, ahead, len, ring + put * R::kBytes, lane);
      there = (there & ~((unsigned long long)all_keys<R>() << (R::kKeys * put))) | (unsigned long long)keys << (R::kKeys * put);
      put = put + 1 == S ? 0 : put + 1;
      const int was = ahead.row;
      if (new_job && win.next_row <= was) {                    // the row after this one
        int r = was + 1;
        while (r < a.rows && before[r + 1] == before[r]) ++r;
        if (r < a.rows) win.ahead(a, r, length_of(r), lane);
      }
      advance(ahead);
      new_job = ahead.k == 0;
    };
    const float scale2 = a.scale * kLog2e;
    R x;
    int from = c.k, head0 = 0, count = 0;
    uint32_t phase = 0;
    bool fresh = true, first = true;
#pragma unroll 1
    for (int lead = S - 1;;) {
      fetch();
      if (lead > 0) {        // the first rounds are on their way before any is waited for
        --lead;
        continue;
      }
      if (c.unit >= w1) break;
      if (fresh) {
        const int tile = c.vh - c.kv * head_tiles;
        head0 = c.kv * group + tile * tile_heads;
        count = min(tile_heads, group - tile * tile_heads);
        from = c.k;
      }
      if constexpr (TMA) mbar_wait(bars + take, phase, &aborted, kWaitFullTimeout);
      if (fresh) {
        x.start(a, my_queries + take_job * R::kQueryBytes, count, lane);
        fresh = false;
      }
      const unsigned keys = (unsigned)(there >> (R::kKeys * take)) & all_keys<R>();
      if (keys != all_keys<R>()) {
        // What lies where no key is may be NaN: a weight of zero times a value of zero instead.
        unsigned char* values = ring + take * R::kBytes + R::kSegs * R::kSeg;
        for (int i = lane; i < R::kSegs * R::kKeys * 8; i += 32)
          if (!(keys >> (i >> 3 & (R::kKeys - 1)) & 1)) reinterpret_cast<uint4*>(values)[i] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();                              // ahead of the copy that reuses the place
        __syncwarp();
      }
      x.compute(smem_u32(ring) + take * R::kBytes, keys, scale2, my_queries + take_job * R::kQueryBytes, lane);
      __syncwarp();
      if (++take == S) {
        take = 0;
        phase ^= 1;
      }
      const bool last = c.k + 1 == c.n;
      const int job_begin = c.unit - c.k;
      const Cursor was = c;
      advance(c);
      if (last || c.unit >= w1) {
        x.finish(lane);
        if (from == 0 && last) {
          T* out = static_cast<T*>(a.o) + was.row * a.o_row + (long long)head0 * a.o_head;
          x.each(lane, [&](int h, int f, const auto& v, float, float l) {
            if (h < count) store_out(out + h * a.o_head + f, v, 1.0f / l, a.hd - f, o_vec);
          });
        } else {
          const int at = 2 * warp + (first ? 0 : 1);
          float* part = first ? leads + warp * kPart : reinterpret_cast<float*>(rings + warp * S * R::kBytes);
          __syncwarp();
          x.each(lane, [&](int h, int f, const auto& v, float m, float l) {
            if (h >= count) return;
            constexpr int N = sizeof(v) / sizeof(float);
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(part + h * R::kHD + f + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            if (f == 0) {
              part[R::kHeads * R::kHD + h] = m;
              part[R::kHeads * (R::kHD + 1) + h] = l;
            }
          });
          if (lane == 0) {
            sh.job[at] = was.row * tiles + was.vh;
            sh.row[at] = was.row;
            sh.head[at] = head0;
            sh.count[at] = count;
            sh.begin[at] = job_begin;
            sh.rounds[at] = was.n;
          }
        }
        fresh = true;
        first = false;
        take_job = take_job + 1 == S ? 0 : take_job + 1;
      }
    }
  }
  __syncthreads();

  join_parts<R, W, S>(a, sh, rings, leads, begin, end, share);
}

// Map of the pages [pages, kv_heads, page, hd]: tiles of 128 bytes of `box` tokens.
static int map_pages(CUtensorMap* map, const PagedAttnArgs& a, const void* base, long long page, long long head, long long tok, int box) {
  const uint64_t e = a.f32 ? 4 : 2;
  const uint64_t dims[4] = {(uint64_t)a.hd, (uint64_t)a.page, (uint64_t)a.kv_heads, (uint64_t)a.pages};
  const uint64_t strides[3] = {tok * e, head * e, page * e};
  const uint32_t boxes[4] = {(uint32_t)(128 / e), (uint32_t)box, 1, 1};
  return encode_tmap_nd(map, a.f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, base, 4, dims, strides, boxes);
}

template <typename R, int W, int S, bool TMA = true>
static int launch_paged(const PagedAttnArgs& a, const PageMaps& maps, bool q_vec, bool o_vec, cudaStream_t st) {
  const size_t smem = 1024 + (size_t)W * S * (R::kBytes + R::kQueryBytes) + W * Part<R>::kFloats * 4 + (a.rows + 1) * 4 + a.rows;
  constexpr int kLimit = 226 << 10;
  static SmemLimit limit;
  const int grid = sm_count();
  if (smem > kLimit || a.ws_floats < grid * 2LL * Part<R>::kFloats || a.num_counters < grid) return kErrTooLarge;
  DPTB_CUDA_OK(limit.raise((const void*)paged_attention_kernel<R, W, S, TMA>, kLimit));
  int box_shift = 0;
  while (2 << box_shift <= R::kKeys && a.page % (2 << box_shift) == 0) ++box_shift;
  paged_attention_kernel<R, W, S, TMA><<<grid, W * 32, smem, st>>>(a, maps, box_shift, (a.heads / a.kv_heads + R::kHeads - 1) / R::kHeads, R::kHeads, q_vec, o_vec);
  return counted(1, (int)cudaGetLastError());
}

}  // namespace dptb

using namespace dptb;

extern "C" int dptb_paged_attention(const PagedAttnArgs* args, void* stream) {
  PagedAttnArgs a = *args;
  if (a.rows == 0 || a.heads == 0) return 0;
  if (a.rows < 0 || a.rows > 65535 || a.heads < 0 || a.kv_heads <= 0 || a.heads % a.kv_heads || a.hd <= 0 || a.hd > kMaxHeadDim ||
      a.page <= 0 || a.width < 0 || a.pages < 0)
    return kErrBadShape;
  a.page_shift = 31;
  while (1LL << (a.page_shift - 31) < a.page) ++a.page_shift;
  a.page_mul = (unsigned)(((1ULL << a.page_shift) + a.page - 1) / a.page);
  auto st = static_cast<cudaStream_t>(stream);
  const int per = a.f32 ? 4 : 8;                       // elements of a piece
  auto whole = [&](const void* p, long long s0, long long s1, long long s2) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % per == 0 && s1 % per == 0 && s2 % per == 0;
  };
  const int keys = a.f32 ? (a.hd <= 64 ? 16 : 8) : a.hd <= 64 ? 32 : 16;
  // rounds, and all else that is counted, in 32 bits
  if ((double)a.rows * ((double)a.width * a.page / keys + 2) * a.heads >= 2147483000.0) return kErrTooLarge;
  const bool qv = whole(a.q, a.q_row, a.q_head, 0), ov = whole(a.o, a.o_row, a.o_head, 0);
  const int group = a.heads / a.kv_heads;
  PageMaps maps = {};
  int box = 1;
  while (2 * box <= keys && a.page % (2 * box) == 0) box *= 2;
  const bool tma = a.hd % per == 0 && whole(a.k, a.k_page, a.k_head, a.k_tok) && whole(a.v, a.v_page, a.v_head, a.v_tok) &&
                   map_pages(&maps.k, a, a.k, a.k_page, a.k_head, a.k_tok, box) == 0 && map_pages(&maps.v, a, a.v, a.v_page, a.v_head, a.v_tok, box) == 0;
#define DPTB_PAGED(...) return launch_paged<__VA_ARGS__>(a, maps, qv, ov, st)
  if (!tma && a.f32) {
    if (a.hd <= 64) DPTB_PAGED(F32Round<64, 4, 4>, 8, 2, false);
    if (a.hd <= 128) DPTB_PAGED(F32Round<128, 4, 2>, 8, 2, false);
    DPTB_PAGED(F32Round<256, 4, 2>, 4, 2, false);
  }
  if (!tma) {
    if (a.hd <= 64) DPTB_PAGED(Bf16Round<64, 1, 2>, 8, 2, false);
    if (a.hd <= 128) DPTB_PAGED(Bf16Round<128, 1, 1>, 8, 2, false);
    DPTB_PAGED(Bf16Round<256, 1, 1>, 4, 2, false);
  }
  if (!a.f32) {
    if (a.hd <= 64 && group <= 8) DPTB_PAGED(Bf16Round<64, 1, 2>, 8, 2);
    if (a.hd <= 64) DPTB_PAGED(Bf16Round<64, 2, 2>, 8, 2);
    if (a.hd <= 128 && group <= 8) DPTB_PAGED(Bf16Round<128, 1, 1>, 8, 2);
    if (a.hd <= 128) DPTB_PAGED(Bf16Round<128, 2, 1>, 6, 2);
    DPTB_PAGED(Bf16Round<256, 1, 1>, 4, 2);
  }
  // Eight warps, fewer where registers or shared memory hold no more; twelve and ten where a round is short, 6 KB (16 sequences of 2048 keys, 8 kv heads
  // of 80: 44 us with eight, 37 with twelve; group of four 53 and 50 with ten).  Of 8 KB rounds eight warps have enough in flight: heads of 128,
  // 64 sequences of 500 keys, 71 us, 73 with eleven.
#define DPTB_PAGED_GROUP(HD, NJ, W, W4) \
  if (group == 1) DPTB_PAGED(F32Round<HD, 1, NJ>, W, 2); \
  if (group == 2) DPTB_PAGED(F32Round<HD, 2, NJ>, W, 2); \
  if (group <= 4) DPTB_PAGED(F32Round<HD, 4, NJ>, W4, 2)
  if (a.hd <= 64) { DPTB_PAGED_GROUP(64, 4, 8, 8); DPTB_PAGED(F32Round<64, 8, 4>, 8, 2); }
  if (a.hd <= 96) { DPTB_PAGED_GROUP(96, 2, 12, 10); DPTB_PAGED(F32Round<96, 8, 2>, 8, 2); }
  if (a.hd <= 128) { DPTB_PAGED_GROUP(128, 2, 8, 8); DPTB_PAGED(F32Round<128, 8, 2>, 7, 2); }
  DPTB_PAGED_GROUP(256, 2, 4, 4);
  DPTB_PAGED(F32Round<256, 4, 2>, 4, 2);
#undef DPTB_PAGED_GROUP
#undef DPTB_PAGED
}
