// Pages of a key / value cache: the append of a step's rows, and the operations on who holds which page.
//
// A cache is a pool of pages, `page` tokens each, and a table that lists the pages of every sequence ("row") in order; -1 stands behind
// the last.  A page may be listed by several rows (beams that share a prompt).  Who holds what is read off the table alone: a page is free
// when no row lists it, so there are no counts that could go wrong, and every operation is a function of the table.
//
// All of it runs on the device without the host's knowledge, so that a decoding loop needs no synchronisation and can be captured.
#include <cuda_bf16.h>
#include <math.h>

#include "common/host.h"
#include "common/ptx.cuh"
#include "common/reduce.cuh"

namespace dptb {

// ------------------------------------------------------------------------------------------------------------ append
// Row t of `qkv` is [Hq | Hkv | Hkv] heads of a token at positions[t] of sequence rows[t].  Queries and keys are turned in half-split
// form, pair (d, d + rotary / 2) by position * base^(-2 d / rotary); keys and values go to their place in the pages.  A token of
// negative position has no place and passes unturned (padding).  The angle, its sine and its cosine are formed in 64 bits and rounded once: in 32
// a position of 100000 leaves the angle 0.004 rad off, and one that is reduced to a turn before it is rounded is off by up to 2^-23.
//
// Bound by memory, or by the launch for a step.  A CTA takes up to four tokens: their angles first, one a thread, into shared memory, then the
// heads in 16-byte groups.  3.6 us for 32 tokens of 32 + 2 x 8 heads of 128 in bf16; 14.5 us where 72 MB move (5.0 TB/s; eight tokens a CTA: 14.7).
struct AppendArgs {
  const void* qkv;
  void* q;                // [tokens, heads, hd], contiguous
  void* keys;             // [tokens, kv_heads, hd], contiguous, or null: the turned keys once more
  void* k;                // pages
  void* v;
  const int* table;
  const int* positions;
  const int* rows;        // null: token t belongs to row t
  long long ld, k_page, k_head, k_tok, v_page, v_head, v_tok, table_row;
  int tokens, heads, kv_heads, hd, rotary, page, width, pages, table_rows, f32;
  double base;            // its logarithm to base 2 in the kernel
};
static_assert(sizeof(AppendArgs) == 176, "packed by the caller");

constexpr int kAppendThreads = 256;
constexpr int kAppendPairs = 128;    // of a head of 256 features
constexpr int kAppendTokens = 4;

// n / d = n * mul >> shift for 0 <= n < 2^31: mul = ceil(2^shift / d) with 2^(shift - 31) >= d, whose excess, less than one, adds less than the
// last place of a quotient.
struct Divisor {
  unsigned mul, shift;
  static Divisor of(int d) {
    Divisor x{0, 31};
    while (1LL << (x.shift - 31) < d) ++x.shift;
    if (d > 0) x.mul = (unsigned)(((1ULL << x.shift) + d - 1) / d);
    return x;
  }
  __device__ __forceinline__ int divide(int n) const { return (int)((unsigned long long)(unsigned)n * mul >> shift); }
};
struct AppendShape {
  Divisor pairs, whole, tail, by_turned, by_kv;      // groups of a half, of a head, behind the turned features; heads
  int tokens;                                        // of a CTA
};

template <typename T, int VEC>
__device__ __forceinline__ void load_group(const T* p, float (&f)[VEC]) {
  T e[VEC];
  if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);
  else e[0] = *p;
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = to_f32(e[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_group(T* p, const float (&f)[VEC]) {
  T e[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(f[i]);
  if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
  else *p = e[0];
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kAppendThreads)
paged_append_kernel(const AppendArgs a, const AppendShape shape) {
  __shared__ float2 turn[kAppendTokens * kAppendPairs];
  __shared__ int page_of[kAppendTokens], off_of[kAppendTokens];
  const int t0 = blockIdx.x * shape.tokens, nt = min(shape.tokens, a.tokens - t0);
  const int tid = threadIdx.x, half = a.rotary / 2, turned = a.heads + a.kv_heads;
  const T* x = static_cast<const T*>(a.qkv) + t0 * a.ld;
  const int pairs = half / VEC, whole = a.hd / VEC, tail = (a.hd - a.rotary) / VEC;
  if (tid < nt) {
    const int pos = a.positions[t0 + tid], row = a.rows ? a.rows[t0 + tid] : t0 + tid;
    int page = -1;
    if (pos >= 0) {
      const int slot = pos / a.page;
      if (row >= 0 && row < a.table_rows && slot < a.width) page = a.table[row * a.table_row + slot];
      if (page < 0 || page >= a.pages) {      // no place for it: nothing is written
        report_error(kBadPage);
        page = -1;
      }
      off_of[tid] = pos - slot * a.page;
    }
    page_of[tid] = page;
  }
  for (int i = tid; i < nt * half; i += kAppendThreads) {
    const int t = i / half, d = i - t * half, pos = a.positions[t0 + t];
    float sn = 0.0f, cs = 1.0f;
    if (pos > 0) {
      constexpr double kHalfTurns = 1.0 / 3.141592653589793238463;
      double s64, c64;
      sincospi(pos * exp2(-2.0 * d / a.rotary * a.base) * kHalfTurns, &s64, &c64);
      sn = (float)s64;
      cs = (float)c64;
    }
    turn[i] = make_float2(cs, sn);
  }
  __syncthreads();
  auto put = [&](int t, int h, int d, const float (&f)[VEC]) {
    const long long tok = t0 + t;
    if (h < a.heads) {
      store_group<T, VEC>(static_cast<T*>(a.q) + (tok * a.heads + h) * a.hd + d, f);
      return;
    }
    const int page = page_of[t], g = h - a.heads;
    if (h < turned) {
      if (a.keys) store_group<T, VEC>(static_cast<T*>(a.keys) + (tok * a.kv_heads + g) * a.hd + d, f);
      if (page >= 0) store_group<T, VEC>(static_cast<T*>(a.k) + page * a.k_page + off_of[t] * a.k_tok + g * a.k_head + d, f);
    } else if (page >= 0) {
      store_group<T, VEC>(static_cast<T*>(a.v) + page * a.v_page + off_of[t] * a.v_tok + (h - turned) * a.v_head + d, f);
    }
  };
  // Several groups' loads are on their way together: the compiler moves none over a store that might change what it reads.
  constexpr int U = 3;
  const int n_pairs = nt * turned * pairs, n_tail = nt * turned * tail, n_whole = nt * a.kv_heads * whole;
  for (int i0 = tid; i0 < n_pairs; i0 += U * kAppendThreads) {
    float lo[U][VEC], hi[U][VEC];
    int t[U], h[U], d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * kAppendThreads, n_pairs - 1), n = shape.pairs.divide(i);
      d[u] = (i - n * pairs) * VEC;
      t[u] = shape.by_turned.divide(n);
      h[u] = n - t[u] * turned;
      const T* src = x + t[u] * a.ld + h[u] * a.hd + d[u];
      load_group<T, VEC>(src, lo[u]);
      load_group<T, VEC>(src + half, hi[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * kAppendThreads >= n_pairs) break;
      const float2* w = turn + t[u] * half + d[u];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float2 c = w[j];
        const float p = lo[u][j] * c.x - hi[u][j] * c.y, q = hi[u][j] * c.x + lo[u][j] * c.y;
        lo[u][j] = p;
        hi[u][j] = q;
      }
      put(t[u], h[u], d[u], lo[u]);
      put(t[u], h[u], half + d[u], hi[u]);
    }
  }
  for (int i = tid; i < n_tail; i += kAppendThreads) {                   // features that are not turned
    const int n = shape.tail.divide(i), d = a.rotary + (i - n * tail) * VEC, t = shape.by_turned.divide(n), h = n - t * turned;
    float f[VEC];
    load_group<T, VEC>(x + t * a.ld + h * a.hd + d, f);
    put(t, h, d, f);
  }
  for (int i = tid; i < n_whole; i += kAppendThreads) {
    const int n = shape.whole.divide(i), d = (i - n * whole) * VEC, t = shape.by_kv.divide(n), h = turned + n - t * a.kv_heads;
    float f[VEC];
    load_group<T, VEC>(x + t * a.ld + h * a.hd + d, f);
    put(t, h, d, f);
  }
}

template <typename T, int VEC>
static int launch_append(AppendArgs a, cudaStream_t st) {
  auto whole = [](const void* p, long long s0, long long s1, long long s2) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s0 % VEC == 0 && s1 % VEC == 0 && s2 % VEC == 0;
  };
  const bool vec = a.hd % VEC == 0 && a.rotary / 2 % VEC == 0 && whole(a.qkv, a.ld, 0, 0) && whole(a.q, 0, 0, 0) &&
                   whole(a.keys, 0, 0, 0) && whole(a.k, a.k_page, a.k_head, a.k_tok) && whole(a.v, a.v_page, a.v_head, a.v_tok);
  const int v = vec ? VEC : 1, half = a.rotary / 2;
  a.base = log2(a.base);
  // At least four CTAs an SM before one takes several tokens.
  const int per = a.tokens / (4 * sm_count());
  const AppendShape shape{Divisor::of(half / v), Divisor::of(a.hd / v), Divisor::of((a.hd - a.rotary) / v), Divisor::of(a.heads + a.kv_heads),
                          Divisor::of(a.kv_heads), per < 1 ? 1 : per > kAppendTokens ? kAppendTokens : per};
  const int grid = (a.tokens + shape.tokens - 1) / shape.tokens;
  if (vec) paged_append_kernel<T, VEC><<<grid, kAppendThreads, 0, st>>>(a, shape);
  else     paged_append_kernel<T, 1><<<grid, kAppendThreads, 0, st>>>(a, shape);
  return counted(1, (int)cudaGetLastError());
}

// ------------------------------------------------------------------------------------------------------------ who holds what
constexpr int kPageThreads = 1024;
constexpr int kMaxForkRows = 4096, kRowBits = 12;
constexpr int kMaxPages = 1 << 19;       // with a row in 31 bits
constexpr int kPageCluster = 8;
constexpr int kPageSmem = 224 << 10;    // both bit maps of the largest pool, and the rows

// Exclusive sum over the block; `total` is everybody's sum.  `scratch`: 33 ints.
__device__ __forceinline__ int block_scan(int v, int* scratch, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = s;
  __syncthreads();
  if (warp == 0) {
    const int w = lane < (int)(blockDim.x >> 5) ? scratch[lane] : 0;
    int t = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    scratch[lane] = t - w;
    if (lane == 31) scratch[32] = t;
  }
  __syncthreads();
  total = scratch[32];
  return scratch[warp] + s - v;
}

__device__ __forceinline__ void mark(unsigned* bits, int page) {
  const unsigned b = 1u << (page & 31);
  if (!(reinterpret_cast<volatile unsigned*>(bits)[page >> 5] & b)) atomicOr(bits + (page >> 5), b);
}

// CTAs of a cluster mark pages in maps of their own; this one's word i joined with the others'.
__device__ __forceinline__ unsigned joined(const unsigned* bits, int i, unsigned ctas) {
  unsigned v = 0;
  for (unsigned c = 0; c < ctas; ++c) {
    unsigned u;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(u) : "r"(map_to_cta(bits + i, c)) : "memory");
    v |= u;
  }
  return v;
}
__device__ __forceinline__ unsigned cluster_ctas() {
  unsigned n;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
  return n;
}

// New row r is row parents[r] of the old table (-1: empty), longer by `grow` tokens.  Pages for these come from the free ones, lowest numbers
// first, in the order of the rows.  The last page of a row that grows into it must be the row's own: it is when no other row lists it but
// such as grow into it too, and the first of these keeps it; the others take a copy, which (src, dst) name for the kernel that copies.
//
// One cluster: the CTAs share the rows, a warp a row, and mark pages in bit maps in shared memory (listed at all; listed by somebody who does not grow
// into it).  The first CTA joins the maps and does what needs all rows: a hash table from a page to the first row that grows into it, and sums over rows and pages
// for the order.  Bound by a chain of a dozen latencies: 4.9 us for four rows of 13 pages, 10 us for 256 rows of 94.
struct ForkArgs {
  const int* table;
  const int* lens;
  const int* parents;     // null: every row itself
  const int* grow;        // null: grow_all for every row that holds tokens
  int* new_table;         // [rows, width]
  int* new_lens;
  int* src;               // [rows]
  int* dst;
  int* free_list;         // [pages] of scratch: the pages to be given
  long long table_row;
  int rows_in, rows, width, pages, page, grow_all;
};
static_assert(sizeof(ForkArgs) == 104, "packed by the caller");

struct ForkRow {
  int parent, old_len, new_len, held, want;
  bool grows;             // into a page that holds tokens already
};

__device__ __forceinline__ ForkRow fork_row(const ForkArgs& a, int r) {
  ForkRow f;
  f.parent = a.parents ? a.parents[r] : r;
  if (f.parent >= a.rows_in) f.parent = -1;
  const long long room = min((long long)a.width * a.page, 0x7fffffffLL);
  f.old_len = f.parent >= 0 ? (int)min((long long)max(a.lens[f.parent], 0), room) : 0;
  const long long more = a.grow ? max(a.grow[r], 0) : f.old_len > 0 ? a.grow_all : 0;
  f.new_len = (int)min(f.old_len + more, room);
  f.held = (f.old_len + a.page - 1) / a.page;
  f.want = (int)(((long long)f.new_len + a.page - 1) / a.page);
  f.grows = f.new_len > f.old_len && f.old_len % a.page != 0;
  return f;
}

__global__ void __launch_bounds__(kPageThreads)
fork_pages_kernel(const ForkArgs a, int words, int slots) {
  extern __shared__ unsigned smem[];
  unsigned* used = smem;                                     // [words]
  unsigned* others = used + words;                           // [words]
  // Of the first CTA:
  unsigned* hash = others + words;                           // [slots]: page and first row that grows into it
  int* tail = reinterpret_cast<int*>(hash + slots);          // [rows]: page that a row grows into, -1 if none
  int* held = tail + a.rows;                                 // [rows]
  int* rank = held + a.rows;                                 // [rows]: pages that a row wants; pages given to the rows before
  __shared__ int scratch[33];
  constexpr unsigned kEmpty = 0xffffffffu;
  const unsigned cta = cluster_cta_rank(), ctas = cluster_ctas();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = kPageThreads / 32;
  for (int i = tid; i < 2 * words; i += kPageThreads) used[i] = 0;
  if (cta == 0)
    for (int i = tid; i < slots; i += kPageThreads) hash[i] = kEmpty;
  cluster_sync_all();                                        // (every CTA has started: its memory can be written)
  for (int r = cta * nw + warp; r < a.rows; r += ctas * nw) {
    const ForkRow f = fork_row(a, r);
    if (lane == 0) {
      const bool bad = a.parents && a.parents[r] >= a.rows_in;
      const long long more = a.grow ? max(a.grow[r], 0) : f.old_len > 0 ? a.grow_all : 0;
      if (bad || f.parent >= 0 && a.lens[f.parent] > f.old_len || f.new_len < f.old_len + more) report_error(kBadPage);
      a.new_lens[r] = f.new_len;
      st_cluster_u32(map_to_cta(held + r, 0), f.held);
      st_cluster_u32(map_to_cta(rank + r, 0), f.want - f.held);
      if (!f.grows) st_cluster_u32(map_to_cta(tail + r, 0), kEmpty);
    }
    const int* row = a.table + (f.parent < 0 ? 0 : f.parent) * a.table_row;
    int* out = a.new_table + (long long)r * a.width;
    for (int s0 = lane; s0 < a.width; s0 += 4 * 32) {
      int page[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) page[x] = s0 + 32 * x < f.held ? row[s0 + 32 * x] : -1;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int s = s0 + 32 * x;
        if (s >= a.width) break;
        if (s < f.held) {
          if ((unsigned)page[x] >= (unsigned)a.pages) {
            report_error(kBadPage);
            page[x] = -1;
          } else {
            mark(used, page[x]);
          }
          if (f.grows && s == f.held - 1) st_cluster_u32(map_to_cta(tail + r, 0), page[x]);
          else if (page[x] >= 0) mark(others, page[x]);
        }
        out[s] = page[x];
      }
    }
  }
  cluster_sync_all();
  if (cta == 0 && ctas > 1)
    for (int i = tid; i < 2 * words; i += kPageThreads) used[i] = joined(used, i, ctas);
  if (ctas > 1) cluster_sync_all();                          // the first CTA has read the others' maps
  if (cta != 0) return;
  __syncthreads();
  auto place = [&](int page) { return (int)((unsigned)page * 2654435761u % (unsigned)slots); };
  for (int r = tid; r < a.rows; r += kPageThreads) {
    const int page = tail[r];
    if (page < 0) continue;
    const unsigned mine = (unsigned)page << kRowBits | (unsigned)r;
    int i = place(page);
    for (int n = 0; n < slots; ++n) {                        // (more slots than rows: it ends)
      const unsigned had = atomicCAS(hash + i, kEmpty, mine);
      if (had == kEmpty) break;
      if (had >> kRowBits == (unsigned)page) {
        atomicMin(hash + i, mine);
        break;
      }
      i = i + 1 == slots ? 0 : i + 1;
    }
  }
  __syncthreads();
  int need_all = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kPageThreads) {
    const int r = r0 + tid;
    int need = 0;
    bool copies = false;
    if (r < a.rows) {
      const int page = tail[r];
      if (page >= 0) {
        int i = place(page);
        while (hash[i] >> kRowBits != (unsigned)page) i = i + 1 == slots ? 0 : i + 1;      // (it is there)
        copies = (others[page >> 5] >> (page & 31) & 1) || (hash[i] & ((1u << kRowBits) - 1)) != (unsigned)r;
      }
      need = rank[r] + copies;
      a.src[r] = a.dst[r] = -1;
    }
    int total;
    const int before = block_scan(need, scratch, total);
    if (r < a.rows) rank[r] = (need_all + before) << 1 | (int)copies;
    need_all += total;
  }
  int found = 0;
  for (int w0 = 0; w0 < words && found < need_all; w0 += kPageThreads) {
    const int w = w0 + tid;
    unsigned open = 0;
    if (w < words) {
      open = ~used[w];
      if ((w + 1) * 32 > a.pages) open &= (1u << (a.pages & 31)) - 1;
    }
    int total;
    int at = found + block_scan(__popc(open), scratch, total);
    for (; open && at < need_all; ++at, open &= open - 1) a.free_list[at] = w * 32 + __ffs(open) - 1;
    found += total;
  }
  __syncthreads();
  if (found < need_all && tid == 0) report_error(kPoolFull);
  for (int k = tid; k < need_all; k += kPageThreads) {       // the k-th page to be given, and whose it is
    int r = 0, hi = a.rows - 1;
    while (r < hi) {
      const int mid = (r + hi + 1) / 2;
      if (rank[mid] >> 1 <= k) r = mid;
      else hi = mid - 1;
    }
    const bool copies = rank[r] & 1;
    const int i = k - (rank[r] >> 1), page = k < found ? a.free_list[k] : -1;
    a.new_table[(long long)r * a.width + held[r] + i - copies] = page;
    if (copies && i == 0 && page >= 0) {
      a.src[r] = tail[r];
      a.dst[r] = page;
    }
  }
}

// The live pages get the lowest numbers: of the n that are listed, those numbered n and above move, in order, to the free numbers below n.
struct CompactArgs {
  const int* table;
  int* new_table;
  int* src;               // [pages / 2]
  int* dst;
  int* live;              // [1]
  long long table_row;
  int rows, width, pages;
};
static_assert(sizeof(CompactArgs) == 64, "packed by the caller");

// One cluster: the CTAs share the rows, each has the joined map, and they share the pages.
__global__ void __launch_bounds__(kPageThreads)
compact_pages_kernel(const CompactArgs a, int words) {
  extern __shared__ unsigned smem[];
  unsigned* mine = smem;                                     // [words]: pages that this CTA's rows list
  unsigned* used = mine + words;                             // [words]: that any lists
  int* before = reinterpret_cast<int*>(used + words);        // [words]: listed pages ahead of a word
  __shared__ int scratch[33];
  const unsigned cta = cluster_cta_rank(), ctas = cluster_ctas();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = kPageThreads / 32;
  for (int i = tid; i < words; i += kPageThreads) mine[i] = 0;
  __syncthreads();
  for (int r = cta * nw + warp; r < a.rows; r += ctas * nw)
    for (int s0 = lane; s0 < a.width; s0 += 4 * 32) {
      int page[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) page[x] = s0 + 32 * x < a.width ? a.table[r * a.table_row + s0 + 32 * x] : -1;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (page[x] >= a.pages) report_error(kBadPage);
        else if (page[x] >= 0) mark(mine, page[x]);
      }
    }
  cluster_sync_all();
  int live = 0;
  for (int w0 = 0; w0 < words; w0 += kPageThreads) {
    const int w = w0 + tid;
    const unsigned bits = w < words ? joined(mine, w, ctas) : 0;
    int total;
    const int at = live + block_scan(__popc(bits), scratch, total);
    if (w < words) {
      used[w] = bits;
      before[w] = at;
    }
    live += total;
  }
  __syncthreads();
  auto rank = [&](int page) { return before[page >> 5] + __popc(used[page >> 5] & ((1u << (page & 31)) - 1)); };
  const int kept = live < a.pages ? rank(live) : live;       // live pages that stay: those below `live`
  const int moves = live - kept, first = cta * kPageThreads + tid, step = ctas * kPageThreads;
  for (int i = first; i < a.pages / 2; i += step) {
    if (i >= moves) a.src[i] = a.dst[i] = -1;
  }
  for (int p = first; p < a.pages; p += step) {
    const bool on = used[p >> 5] >> (p & 31) & 1;
    if (p < live && !on) a.dst[p - rank(p)] = p;
    if (p >= live && on) a.src[rank(p) - kept] = p;
  }
  if (first == 0) *a.live = live;
  cluster_sync_all();                                        // dst is there, and nobody reads another's map any more
  for (int r = cta * nw + warp; r < a.rows; r += ctas * nw)
    for (int s0 = lane; s0 < a.width; s0 += 4 * 32) {
      int page[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) page[x] = s0 + 32 * x < a.width ? a.table[r * a.table_row + s0 + 32 * x] : -1;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        if (page[x] < 0 || page[x] >= a.pages) page[x] = -1;
        else if (page[x] >= live) page[x] = __ldcg(a.dst + rank(page[x]) - kept);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (s0 + 32 * x < a.width) a.new_table[(long long)r * a.width + s0 + 32 * x] = page[x];
    }
}

// Up to 32 rows a CTA has a warp for each; more are shared by a cluster (a fork of 4 rows takes 4.9 to 5.7 us in one CTA and 6.1 in eight, of 32 rows of
// 94 pages 7.3 and 7.9, of 64 9.8 and 8.4, of 256 23 and 10).
template <typename... KArgs>
static int launch_page_kernel(void (*kernel)(KArgs...), SmemLimit& limit, int rows, size_t smem, cudaStream_t st, KArgs... args) {
  if (smem > kPageSmem) return kErrTooLarge;
  DPTB_CUDA_OK(limit.raise((const void*)kernel, kPageSmem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows <= 32 ? 1 : kPageCluster);
  cfg.blockDim = dim3(kPageThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cfg.gridDim.x;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return counted(1, (int)cudaLaunchKernelEx(&cfg, kernel, args...));
}

// pool[o, dst[i]] = pool[o, src[i]] for every o < outer and every i with a src, `bytes` a page.  Nobody's dst is somebody's src.
struct CopyArgs {
  void* pool;
  const int* src;
  const int* dst;
  long long outer, bytes;
  int n, pages;
};
static_assert(sizeof(CopyArgs) == 48, "packed by the caller");

constexpr int kCopyThreads = 256;
template <typename V>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(unsigned char* pool, const int* __restrict__ src, const int* __restrict__ dst, int n, int pages, long long bytes) {
  unsigned char* base = pool + blockIdx.y * (long long)pages * bytes;
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int from = src[i], to = dst[i];
    if (from < 0 || to < 0) continue;
    if (from >= pages || to >= pages) {
      if (threadIdx.x == 0) report_error(kBadPage);
      continue;
    }
    const V* x = reinterpret_cast<const V*>(base + from * bytes);
    V* y = reinterpret_cast<V*>(base + to * bytes);
    const int count = (int)(bytes / (long long)sizeof(V));
    for (int j = threadIdx.x; j < count; j += 4 * kCopyThreads) {
      V v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u * kCopyThreads < count) v[u] = x[j + u * kCopyThreads];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + u * kCopyThreads < count) y[j + u * kCopyThreads] = v[u];
    }
  }
}

}  // namespace dptb

using namespace dptb;

extern "C" int dptb_paged_append(const AppendArgs* args, void* stream) {
  const AppendArgs& a = *args;
  if (a.tokens == 0) return 0;
  if (a.tokens < 0 || a.heads < 0 || a.kv_heads <= 0 || a.hd <= 0 || a.hd > 2 * kAppendPairs || a.rotary < 0 || a.rotary % 2 ||
      a.rotary > a.hd || a.page <= 0 || a.width < 0 || a.pages < 0)
    return kErrBadShape;
  auto st = static_cast<cudaStream_t>(stream);
  return a.f32 ? launch_append<float, 4>(a, st) : launch_append<__nv_bfloat16, 8>(a, st);
}

extern "C" int dptb_fork_pages(const ForkArgs* args, void* stream) {
  const ForkArgs& a = *args;
  if (a.rows == 0) return 0;
  if (a.rows < 0 || a.rows > kMaxForkRows || a.rows_in < 0 || a.width < 0 || a.pages < 0 || a.pages > kMaxPages || a.page <= 0 ||
      a.grow_all < 0)
    return kErrBadShape;
  const int words = (a.pages + 31) / 32, slots = 2 * a.rows;
  static SmemLimit limit;
  return launch_page_kernel(fork_pages_kernel, limit, a.rows, (2 * (size_t)words + (size_t)slots + 3 * (size_t)a.rows) * 4,
                            static_cast<cudaStream_t>(stream), a, words, slots);
}

extern "C" int dptb_compact_pages(const CompactArgs* args, void* stream) {
  const CompactArgs& a = *args;
  if (a.rows < 0 || a.width < 0 || a.pages < 0 || a.pages > kMaxPages) return kErrBadShape;
  const int words = (a.pages + 31) / 32;
  static SmemLimit limit;
  return launch_page_kernel(compact_pages_kernel, limit, a.rows, 3 * (size_t)words * 4, static_cast<cudaStream_t>(stream), a, words);
}

extern "C" int dptb_copy_pages(const CopyArgs* args, void* stream) {
  const CopyArgs& a = *args;
  if (a.n == 0 || a.outer == 0 || a.bytes == 0) return 0;
  if (a.n < 0 || a.outer < 0 || a.outer > 65535 || a.pages < 0 || a.bytes < 0 || a.bytes > 0x7fffffff) return kErrBadShape;
  const dim3 grid(min(a.n, 8 * sm_count()), (unsigned)a.outer);
  auto st = static_cast<cudaStream_t>(stream);
  auto* p = static_cast<unsigned char*>(a.pool);
  if (((reinterpret_cast<uintptr_t>(p) | (uintptr_t)a.bytes) & 15) == 0)
    copy_pages_kernel<uint4><<<grid, kCopyThreads, 0, st>>>(p, a.src, a.dst, a.n, a.pages, a.bytes);
  else
    copy_pages_kernel<unsigned short><<<grid, kCopyThreads, 0, st>>>(p, a.src, a.dst, a.n, a.pages, a.bytes);
  return counted(1, (int)cudaGetLastError());
}
