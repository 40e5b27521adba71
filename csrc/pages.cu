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
// negative position has no place and passes unturned (padding).  The angle is formed and reduced to one turn in 64 bits: in 32 a position of
// 100000 leaves it 0.004 rad off.
//
// Bound by memory, or by the launch for a step.  A CTA takes up to 8 tokens: their angles first, one a thread, into shared memory, then the
// heads by in 16-byte groups.
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
constexpr int kAppendTokens = 8;

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
  const int tid = threadIdx.x, half = a.rotary / 2;
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
      constexpr double kTurn = 6.283185307179586476925, kTurns = 1.0 / kTurn;
      const double turns = pos * exp2(-2.0 * d / a.rotary * a.base) * kTurns;
      sincosf((float)((turns - rint(turns)) * kTurn), &sn, &cs);
    }
    turn[i] = make_float2(cs, sn);
  }
  __syncthreads();
  const int turned = a.heads + a.kv_heads;
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
  const T* x = static_cast<const T*>(a.qkv) + t0 * a.ld;
  const int pairs = half / VEC, whole = a.hd / VEC, tail = (a.hd - a.rotary) / VEC;
#pragma unroll 2
  for (int i = tid; i < nt * turned * pairs; i += kAppendThreads) {
    const int n = shape.pairs.divide(i), d = (i - n * pairs) * VEC, t = shape.by_turned.divide(n), h = n - t * turned;
    const T* src = x + t * a.ld + h * a.hd + d;
    const float2* w = turn + t * half + d;
    float lo[VEC], hi[VEC];
    load_group<T, VEC>(src, lo);
    load_group<T, VEC>(src + half, hi);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float2 c = w[j];
      const float p = lo[j] * c.x - hi[j] * c.y, q = hi[j] * c.x + lo[j] * c.y;
      lo[j] = p;
      hi[j] = q;
    }
    put(t, h, d, lo);
    put(t, h, half + d, hi);
  }
  if (tail > 0)
    for (int i = tid; i < nt * turned * tail; i += kAppendThreads) {     // features that are not turned
      const int n = shape.tail.divide(i), d = a.rotary + (i - n * tail) * VEC, t = shape.by_turned.divide(n), h = n - t * turned;
      float f[VEC];
      load_group<T, VEC>(x + t * a.ld + h * a.hd + d, f);
      put(t, h, d, f);
    }
#pragma unroll 2
  for (int i = tid; i < nt * a.kv_heads * whole; i += kAppendThreads) {
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
constexpr int kMaxForkRows = 4096;
constexpr int kMaxPages = 1 << 19;
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

// New row r is row parents[r] of the old table (-1: empty), longer by `grow` tokens.  Pages for these come from the free ones, lowest numbers
// first, in the order of the rows.  The last page of a row that grows into it must be the row's own: it is when no other row lists it but
// such as grow into it too, and the first of these keeps it; the others take a copy, which (src, dst) name for the kernel that copies.
//
// One CTA: bit maps of the pages in shared memory (listed at all; listed by somebody who does not grow into it), a hash table from a page to the first
// row that grows into it, and sums over rows and pages for the order.
struct ForkArgs {
  const int* table;
  const int* lens;
  const int* parents;     // null: every row itself
  const int* grow;        // null: grow_all for every row that has a parent
  int* new_table;         // [rows, width]
  int* new_lens;
  int* src;               // [rows]
  int* dst;
  int* free_list;         // [pages] of scratch
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
  const long long more = a.grow ? max(a.grow[r], 0) : f.parent >= 0 ? a.grow_all : 0;
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
  int* key = reinterpret_cast<int*>(others + words);         // [slots]: pages that rows grow into
  int* first = key + slots;                                  // [slots]: the lowest such row
  int* rank = first + slots;                                 // [rows]: pages given to the rows before
  __shared__ int scratch[33];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = kPageThreads / 32;
  for (int i = tid; i < 2 * words; i += kPageThreads) used[i] = 0;
  for (int i = tid; i < slots; i += kPageThreads) {
    key[i] = -1;
    first[i] = 0x7fffffff;
  }
  __syncthreads();
  auto find = [&](int page) {
    int i = (int)((unsigned)page * 2654435761u % (unsigned)slots);
    for (int n = 0; n < slots; ++n) {                        // (more slots than rows: it ends)
      const int had = atomicCAS(key + i, -1, page);
      if (had == -1 || had == page) return i;
      i = i + 1 == slots ? 0 : i + 1;
    }
    return 0;
  };
  for (int r = warp; r < a.rows; r += nw) {
    const ForkRow f = fork_row(a, r);
    if (lane == 0) {
      const bool bad = a.parents && a.parents[r] >= a.rows_in;
      const long long more = a.grow ? max(a.grow[r], 0) : f.parent >= 0 ? a.grow_all : 0;
      if (bad || f.parent >= 0 && a.lens[f.parent] > f.old_len || f.new_len < f.old_len + more) report_error(kBadPage);
    }
    const int* row = a.table + (f.parent < 0 ? 0 : f.parent) * a.table_row;
    for (int s = lane; s < a.width; s += 32) {
      int page = -1;
      if (s < f.held) {
        page = row[s];
        if (page < 0 || page >= a.pages) {
          report_error(kBadPage);
          page = -1;
        } else {
          mark(used, page);
          if (f.grows && s == f.held - 1) atomicMin(first + find(page), r);
          else mark(others, page);
        }
      }
      a.new_table[(long long)r * a.width + s] = page;
    }
  }
  __syncthreads();
  int need_all = 0;
  for (int r0 = 0; r0 < a.rows; r0 += kPageThreads) {
    const int r = r0 + tid;
    int need = 0;
    bool copies = false;
    if (r < a.rows) {
      const ForkRow f = fork_row(a, r);
      if (f.grows) {
        const int page = a.new_table[(long long)r * a.width + f.held - 1];
        copies = page >= 0 && ((others[page >> 5] >> (page & 31) & 1) || first[find(page)] != r);
      }
      need = f.want - f.held + copies;
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
  for (int r = warp; r < a.rows; r += nw) {
    const ForkRow f = fork_row(a, r);
    const bool copies = rank[r] & 1;
    const int at = rank[r] >> 1;
    int* row = a.new_table + (long long)r * a.width;
    for (int s = f.held + lane; s < f.want; s += 32) {
      const int i = at + copies + s - f.held;
      row[s] = i < found ? a.free_list[i] : -1;
    }
    if (lane == 0) {
      int from = -1, to = -1;
      if (copies) {
        if (at < found) {
          from = row[f.held - 1];
          to = a.free_list[at];
        }
        row[f.held - 1] = to;
      }
      a.src[r] = from;
      a.dst[r] = to;
      a.new_lens[r] = f.new_len;
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

__global__ void __launch_bounds__(kPageThreads)
compact_pages_kernel(const CompactArgs a, int words) {
  extern __shared__ unsigned smem[];
  unsigned* used = smem;                                     // [words]
  int* before = reinterpret_cast<int*>(used + words);        // [words]: listed pages ahead of a word
  __shared__ int scratch[33];
  const int tid = threadIdx.x;
  for (int i = tid; i < words; i += kPageThreads) used[i] = 0;
  __syncthreads();
  const long long entries = (long long)a.rows * a.width;
  for (long long i = tid; i < entries; i += kPageThreads) {
    const int page = a.table[i / a.width * a.table_row + i % a.width];
    if (page >= a.pages) report_error(kBadPage);
    else if (page >= 0) mark(used, page);
  }
  __syncthreads();
  int live = 0;
  for (int w0 = 0; w0 < words; w0 += kPageThreads) {
    const int w = w0 + tid;
    int total;
    const int at = live + block_scan(w < words ? __popc(used[w]) : 0, scratch, total);
    if (w < words) before[w] = at;
    live += total;
  }
  __syncthreads();
  auto rank = [&](int page) { return before[page >> 5] + __popc(used[page >> 5] & ((1u << (page & 31)) - 1)); };
  const int kept = live < a.pages ? rank(live) : live;       // live pages that stay: those below `live`
  const int moves = live - kept;
  for (int i = tid; i < a.pages / 2; i += kPageThreads) {
    if (i >= moves) a.src[i] = a.dst[i] = -1;
  }
  for (int p = tid; p < a.pages; p += kPageThreads) {
    const bool on = used[p >> 5] >> (p & 31) & 1;
    if (p < live && !on) a.dst[p - rank(p)] = p;
    if (p >= live && on) a.src[rank(p) - kept] = p;
  }
  __syncthreads();
  for (long long i = tid; i < entries; i += kPageThreads) {
    int page = a.table[i / a.width * a.table_row + i % a.width];
    if (page < 0 || page >= a.pages) page = -1;
    else if (page >= live) page = a.dst[rank(page) - kept];
    a.new_table[i] = page;
  }
  if (tid == 0) *a.live = live;
}

// pool[o, dst[i]] = pool[o, src[i]] for every o < outer and every i with a src, `bytes` a page.  Nobody's dst is somebody's src.
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
    for (long long j = threadIdx.x; j < bytes / (long long)sizeof(V); j += kCopyThreads) y[j] = x[j];
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
  const size_t smem = (2 * (size_t)words + 2 * (size_t)slots + a.rows) * 4;
  static SmemLimit limit;
  if (smem > kPageSmem) return kErrTooLarge;
  DPTB_CUDA_OK(limit.raise((const void*)fork_pages_kernel, kPageSmem));
  fork_pages_kernel<<<1, kPageThreads, smem, static_cast<cudaStream_t>(stream)>>>(a, words, slots);
  return counted(1, (int)cudaGetLastError());
}

extern "C" int dptb_compact_pages(const CompactArgs* args, void* stream) {
  const CompactArgs& a = *args;
  if (a.rows < 0 || a.width < 0 || a.pages < 0 || a.pages > kMaxPages) return kErrBadShape;
  const int words = (a.pages + 31) / 32;
  const size_t smem = 2 * (size_t)words * 4;
  static SmemLimit limit;
  if (smem > kPageSmem) return kErrTooLarge;
  DPTB_CUDA_OK(limit.raise((const void*)compact_pages_kernel, kPageSmem));
  compact_pages_kernel<<<1, kPageThreads, smem, static_cast<cudaStream_t>(stream)>>>(a, words);
  return counted(1, (int)cudaGetLastError());
}

extern "C" int dptb_copy_pages(void* pool, const int* src, const int* dst, int n, long long outer, int pages, long long bytes,
                               void* stream) {
  if (n == 0 || outer == 0 || bytes == 0) return 0;
  if (n < 0 || outer < 0 || outer > 65535 || pages < 0 || bytes < 0) return kErrBadShape;
  const dim3 grid(n < 8 * 148 ? n : 8 * 148, (unsigned)outer);
  auto st = static_cast<cudaStream_t>(stream);
  auto* p = static_cast<unsigned char*>(pool);
  if (((reinterpret_cast<uintptr_t>(pool) | (uintptr_t)bytes) & 15) == 0)
    copy_pages_kernel<uint4><<<grid, kCopyThreads, 0, st>>>(p, src, dst, n, pages, bytes);
  else
    copy_pages_kernel<unsigned short><<<grid, kCopyThreads, 0, st>>>(p, src, dst, n, pages, bytes);
  return counted(1, (int)cudaGetLastError());
}
