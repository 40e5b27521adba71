// Beam search's selection: of all continuations of an item's beams, the best as many as it has beams.
//
//   total[b, w, v] = score[b, w] + logit[b * W + w, v] - log sum_u exp(logit[b * W + w, u])
//
// Candidates are ranked by (total, then the lower beam, then the larger logit, then the lower token).  A finished beam has one continuation, `eos` at its old score; its others, those
// of a beam whose score is not finite, and those of a row of logits without a distribution (a NaN, an infinity, nothing but
// -inf) are worth -inf.  Within a beam the order is that of the logits themselves, so that no rounding decides it; totals of different beams
// meet in 64 bits.
//
// beam_kernel: a row is dealt to warps.  One pass over the logits keeps a running maximum and sum of exponentials in every lane; that is
// all that is done for each logit (5.5 instructions in bf16).  The last of an item's CTAs to finish (a counter, no waiting) sums up its rows,
// and the lanes' maxima tell where to look: the best W continuations lie with the lanes of the W largest (each counted with its beam's score),
// and only these lanes' logits are read once more, by the value of the W-th.  That is a few hundred logits, whatever the vocabulary.
//
// Bound by memory for many rows, by a chain of latencies for few.  256 rows of 128256 logits in bf16, 8 beams an item, take 22.7 us, of which the pass is half
// (66 MB in 9 to 11 us) and the choice in each item's last CTA the other; four rows of 50257 in fp32 9.3 us, 35 of 321 7.3.  Choosing in every warp, or in CTAs barrier
// after barrier, cost more than the pass itself: 45 and 61 us for the 256 rows.
#include <cuda_bf16.h>

#include "common/host.h"
#include "common/reduce.cuh"

namespace dptb {

constexpr int kMaxBeams = 32;
constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;
constexpr int kWarpPool = 128;         // candidates of a warp that are ranked at once
constexpr int kItemPool = 1024;        // and of an item
constexpr int kHotLanes = 256;         // lanes whose logits are read again
constexpr int kMaxLists = 64;          // parts of a row
constexpr int kHeld = 5;               // times four lanes' maxima that a thread holds where the choice is made
__host__ __device__ constexpr int mates_of(int beams) { return beams <= 1 ? 8 : beams <= 2 ? 4 : beams <= 4 ? 2 : 1; }      // warps of a row there
constexpr float kLog2e = 1.4426950408889634f;

struct BeamArgs {
  const void* logits;            // [items * beams, ld]
  const float* scores;           // [items, beams]
  const unsigned char* finished; // [items, beams] or null
  float* out_scores;
  int* out_parents;              // row of the parent
  long long* out_tokens;
  unsigned char* out_finished;
  void* ws;                      // BeamPart of every row and warp
  unsigned* counters;            // a zeroed word per item of a launch; zero again afterwards
  long long ld, ws_bytes;
  int items, beams, vocab, eos, f32, num_counters;
  int chunk, lists, vec, first_item;   // set by the launcher: logits of a warp, warps of a row
};
static_assert(sizeof(BeamArgs) == 128, "packed by the caller");

// Larger for a larger value, then for a lower index; zeros of both signs are one value.
__device__ __forceinline__ unsigned long long rank_key(float x, int index) {
  const unsigned u = __float_as_uint(x + 0.0f);
  const unsigned up = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (unsigned long long)up << 32 | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const unsigned up = (unsigned)(key >> 32);
  return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ int key_index(unsigned long long key) { return (int)(0xffffffffu - (unsigned)key); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Descending over the lanes.
__device__ __forceinline__ float sort_lanes(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int j = n >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, j);
      v = ((lane & j) == 0) == ((lane & n) == 0) ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}
// The k-th largest of the block's values, k <= 32: warps sort theirs, and lists are merged pairwise, the 32 largest of two at a time.
__device__ __forceinline__ float kth_largest(float v, int k, float* lists) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = sort_lanes(v);
  lists[warp * 32 + lane] = v;
  __syncthreads();
#pragma unroll 1
  for (int half = kBeamWarps / 2; half > 0; half >>= 1) {
    if (warp < half) {
      v = fmaxf(v, lists[(warp + half) * 32 + 31 - lane]);
#pragma unroll
      for (int j = 16; j > 0; j >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, j);
        v = (lane & j) == 0 ? fmaxf(v, o) : fminf(v, o);
      }
      lists[warp * 32 + lane] = v;
    }
    __syncthreads();
  }
  return lists[k - 1];
}

// 16 bytes of a row.
template <typename T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int N = 4;
  uint32_t u[4];
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(u[i]); }
  __device__ __forceinline__ float top() const { return fmaxf(fmaxf(at(0), at(1)), fmaxf(at(2), at(3))); }
};
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  uint32_t u[4];
  __device__ __forceinline__ float at(int i) const { return __uint_as_float(i & 1 ? u[i >> 1] & 0xffff0000u : u[i >> 1] << 16); }
  __device__ __forceinline__ float top() const {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = reinterpret_cast<const __nv_bfloat162*>(u)[i];
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
  }
};
// Elements first .. first + N of a row of `end`; those beyond are -inf.
__device__ __noinline__ uint4 edge_bits(const unsigned short* row, int first, int end) {      // bf16
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = first + i < end ? row[first + i] : 0xff80u;
  return make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
}
__device__ __noinline__ uint4 edge_bits(const uint32_t* row, int first, int end) {            // fp32
  uint32_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = first + i < end ? row[first + i] : 0xff800000u;
  return make_uint4(e[0], e[1], e[2], e[3]);
}
template <typename T>
__device__ __forceinline__ Piece<T> load_edge(const T* row, int first, int end) {
  uint4 u;
  if constexpr (sizeof(T) == 2) u = edge_bits(reinterpret_cast<const unsigned short*>(row), first, end);
  else u = edge_bits(reinterpret_cast<const uint32_t*>(row), first, end);
  return Piece<T>{u.x, u.y, u.z, u.w};
}
template <typename T>
__device__ __forceinline__ Piece<T> load_whole(const T* row, int first) {
  const uint4 u = *reinterpret_cast<const uint4*>(row + first);
  return Piece<T>{u.x, u.y, u.z, u.w};
}
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* row, int first, int end, bool vec) {
  if (vec && first + Piece<T>::N <= end) return load_whole<T>(row, first);
  if (first < end) return load_edge<T>(row, first, end);
  constexpr uint32_t kNone = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  return Piece<T>{kNone, kNone, kNone, kNone};
}
// What lane `lane` has of the 32 N logits from `first` on: neighbours if rows are on 16-byte boundaries, every 32nd if not, so that a warp's
// loads are whole lines in either case.
template <typename T>
__device__ __forceinline__ int place_in(int first, int lane, int e, bool vec) { return vec ? first + lane * Piece<T>::N + e : first + e * 32 + lane; }
template <typename T, bool VEC>
__device__ __forceinline__ Piece<T> load_group(const T* row, int first, int lane, int end) {
  constexpr int N = Piece<T>::N;
  if constexpr (VEC) return load_piece<T>(row, first + lane * N, end, true);
  const int i = first + lane;
  Piece<T> p;
  if constexpr (sizeof(T) == 2) {
    const auto* bits = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const uint32_t lo = i + e * 32 < end ? bits[i + e * 32] : 0xff80u, hi = i + e * 32 + 32 < end ? bits[i + e * 32 + 32] : 0xff80u;
      p.u[e / 2] = lo | hi << 16;
    }
  } else {
    const auto* bits = reinterpret_cast<const uint32_t*>(row);
#pragma unroll
    for (int e = 0; e < N; ++e) p.u[e] = i + e * 32 < end ? bits[i + e * 32] : 0xff800000u;
  }
  return p;
}

// What a warp leaves of its logits: the sum of exponentials, what it is relative to, every lane's maximum.
struct BeamPart {
  double sum, base;
  float shift, best, pad[2];     // `base` in whole powers of two, NaN where it is none; the largest logit
  float high[32];
};

struct BeamShared {
  unsigned long long keys[kItemPool];      // each warp's kWarpPool; of an item: (beam, token)
  double totals[kItemPool];
  unsigned orders[kItemPool];              // a continuation's logit, larger for a larger one; 0 where its beam does not go by logits
  float lists[kBeamThreads];
  double score[kMaxBeams], top[kMaxBeams], norm[kMaxBeams];
  float size[kMaxBeams];                   // of what fp32 totals are made of
  unsigned char kind[kMaxBeams], fin[kMaxBeams];     // 0: by its logits, 1: finished, 2: nothing to offer; whether finished
  float from[kMaxBeams], least[kMaxBeams];  // what a logit less `from` has to reach
  int hot[kHotLanes], count, hots, counts[kBeamWarps], last;
};
static_assert(kBeamWarps * kWarpPool <= kItemPool, "the warps' pools");

// A sum relative to the maximum `m`, or its shift, relative to `top` > m, or its.
constexpr float kLarge = 1048576.0f;
constexpr double kLn2 = 1.0 / (double)kLog2e;      // of the rounded kLog2e
__device__ __noinline__ double rescaled_large(double s, float m, float shift, float top, float next) {
  const double from = fabsf(m) < kLarge ? (double)shift * kLn2 : (double)m, to = fabsf(top) < kLarge ? (double)next * kLn2 : (double)top;
  return s * exp(from - to);
}
__device__ __forceinline__ double rescaled(double s, float m, float shift, float top, float next) {
  if (m == top || m == -INFINITY) return s;       // (nothing but -inf so far: a sum of 0, or NaN)
  if (fabsf(m) < kLarge && fabsf(top) < kLarge) return next - shift > 1000.0f ? 0.0 * s : s * __longlong_as_double((long long)(1023 + (int)(shift - next)) << 52);
  return rescaled_large(s, m, shift, top, next);
}

// A continuation by its beam's logits.
__device__ __forceinline__ double total_of(const BeamShared& sh, int w, float x) {
  return sh.score[w] + ((double)x - sh.top[w] - sh.norm[w]);      // (a row masked by the lowest value loses nothing to its size)
}
// Continuation i, best first, of a beam that does not go by its logits.
__device__ __forceinline__ double special(const BeamArgs& a, const BeamShared& sh, int w, int i, int& token) {
  token = i;
  if (sh.kind[w] != 1 || a.eos < 0) return -INFINITY;
  token = i == 0 ? a.eos : i - 1 + (i - 1 >= a.eos);      // eos, then the others
  return i == 0 ? sh.score[w] : -INFINITY;
}

// Of a row of logits the best K as keys in `out`, best first, 0 behind the last; by a warp.  The threshold is the K-th largest of the lanes' maxima: what is above
// it lies with fewer than K lanes; of what equals it the first are wanted, in lists where a lane reaches it, and each such list has one or
// is among the fewer than K that have more.  So a masked or flat row is not read again from end to end.
template <typename T>
__device__ __noinline__ void best_of_row(const BeamArgs& a, const T* row, const BeamPart* p, unsigned long long* out, unsigned long long* keys, int* count) {
  constexpr int N = Piece<T>::N;
  const int lane = threadIdx.x & 31, K = a.beams;
  // Lists are looked at eight at a time, a trip to memory each eight: the K-th of all, then the lists with something above it, or at it.
  constexpr int B = 8;
  static_assert(B * 32 * sizeof(float) <= kWarpPool * sizeof(keys[0]) && kMaxLists <= 64, "");
  float* highs = reinterpret_cast<float*>(keys);
  float best = -INFINITY, limit = -INFINITY;      // the 32 largest, descending; the K-th
  auto load = [&](int l0, float (&v)[B]) {
#pragma unroll
    for (int u = 0; u < B; ++u) v[u] = l0 + u < a.lists ? __ldcg(&p[l0 + u].high[lane]) : -INFINITY;
  };
#pragma unroll 1
  for (int l0 = 0; l0 < a.lists; l0 += B) {
    float v[B];
    load(l0, v);
    __syncwarp();
#pragma unroll
    for (int u = 0; u < B; ++u) highs[u * 32 + lane] = v[u];
#pragma unroll 1
    for (int u = 0; u < B; ++u) {
      const float x = highs[u * 32 + lane];
      if (!__any_sync(0xffffffffu, x > limit)) continue;
      best = fmaxf(best, __shfl_sync(0xffffffffu, sort_lanes(x), 31 - lane));
#pragma unroll
      for (int j = 16; j > 0; j >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, best, j);
        best = (lane & j) == 0 ? fmaxf(best, o) : fminf(best, o);
      }
      limit = __shfl_sync(0xffffffffu, best, K - 1);
    }
  }
  unsigned long long over = 0, at_least = 0;      // a bit for each list
#pragma unroll 1
  for (int l0 = 0; l0 < a.lists; l0 += B) {
    float v[B];
    load(l0, v);
#pragma unroll
    for (int u = 0; u < B; ++u) {
      over |= (unsigned long long)(__any_sync(0xffffffffu, v[u] > limit) != 0) << (l0 + u);
      at_least |= (unsigned long long)(l0 + u < a.lists && __any_sync(0xffffffffu, v[u] >= limit)) << (l0 + u);
    }
  }
  if (lane == 0) *count = 0;
  __syncwarp();
#pragma unroll 1
  for (; over; over &= over - 1) {
    const int l = __ffsll(over) - 1, begin = l * a.chunk, end = min(a.vocab, begin + a.chunk);
#pragma unroll 1
    for (unsigned some = __ballot_sync(0xffffffffu, __ldcg(&p[l].high[lane]) > limit); some; some &= some - 1) {
      const int j = __ffs(some) - 1;
#pragma unroll 1
      for (int i = begin + 32 * lane * N; i < end; i += 32 * 32 * N) {
        const Piece<T> x = a.vec ? load_group<T, true>(row, i, j, end) : load_group<T, false>(row, i, j, end);
        if (!(x.top() > limit)) continue;
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (x.at(e) > limit) {
            const int at = atomicAdd(count, 1);
            if (at < kWarpPool) keys[at] = rank_key(x.at(e), place_in<T>(i, j, e, a.vec));
          }
      }
    }
  }
  __syncwarp();
  const int above = *(volatile int*)count;
  if (above > kWarpPool - K) {       // very many with few lanes: the best, one after the other
    unsigned long long last = ~0ull;
#pragma unroll 1
    for (int k = 0; k < K; ++k) {
      unsigned long long top = 0;
      for (int i = lane; i < a.vocab; i += 32) {
        const unsigned long long key = rank_key(to_f32(row[i]), i);
        if (key < last && key > top) top = key;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) out[k] = top;
      last = top;
    }
    return;
  }
  int n = above;
#pragma unroll 1
  for (; at_least && n - above < K; at_least &= at_least - 1) {
    const int l = __ffsll(at_least) - 1, begin = l * a.chunk, end = min(a.vocab, begin + a.chunk);
#pragma unroll 1
    for (int i0 = begin; i0 < end && n - above < K; i0 += 32 * N) {
      const int i = i0 + lane * N;
      const Piece<T> x = load_piece<T>(row, i, end, a.vec);
      int equal = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) equal += i + e < end && x.at(e) == limit;
      int at = equal;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += u;
      }
      const int total = __shfl_sync(0xffffffffu, at, 31);
      at += n - equal;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e < end && x.at(e) == limit) {
          if (at - above < K) keys[at] = rank_key(limit, i + e);
          ++at;
        }
      n += total;
    }
  }
  n = min(n, above + K);
  __syncwarp();
  for (int i = lane; i < n; i += 32) {
    const unsigned long long key = keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > key;
    if (rank < K) out[rank] = key;
  }
  for (int i = n + lane; i < K; i += 32) out[i] = 0;
}

// Where too many are equal, or fewer lanes than beams have anything to offer (a masked vocabulary): the best of every row first.  (64 items of 32 beams over
// 32000 logits that are all the same: 147 us in bf16 and 157 in fp32, 52 and 64 for random ones; with all K K ranked against one another it was 360.)
template <typename T>
__device__ __noinline__ void best_of_rows(const BeamArgs& a, BeamShared& sh, const T* rows, const BeamPart* parts) {
  const int tid = threadIdx.x, warp = tid >> 5, K = a.beams;
  auto* keys = reinterpret_cast<unsigned long long*>(sh.totals);
#pragma unroll 1
  for (int w = warp; w < K; w += kBeamWarps) {
    __syncwarp();
    if (sh.kind[w] == 0) best_of_row<T>(a, rows + w * a.ld, parts + w * a.lists, keys + w * K, sh.keys + warp * kWarpPool, sh.counts + warp);
  }
  __syncthreads();
  for (int c = tid; c < K * K; c += kBeamThreads) {
    const int w = c / K, i = c - w * K;
    const unsigned long long key = keys[c];
    int token = 0;
    double total = -INFINITY;
    bool valid;
    if (sh.kind[w]) {
      valid = i < min(K, a.vocab);
      total = special(a, sh, w, i, token);
    } else {
      valid = key != 0;
      token = key_index(key);
      if (valid) total = total_of(sh, w, key_value(key));
    }
    sh.totals[c] = total;
    sh.keys[c] = valid ? (unsigned long long)w << 32 | (unsigned)token : ~0ull;
  }
  __syncthreads();
}

// The sum of a row's parts: what its logits are taken relative to, and the logarithm of the sum (not finite: no distribution).  The largest logit's own
// term is taken out as it was put in and stands for 1, so that a row of one token is worth nothing but its score and no row more.
__device__ __forceinline__ void sum_row(const BeamPart* p, int lists, double& top, double& norm) {
  const int lane = threadIdx.x & 31;
  double base[2], sum[2], t = 0.0;
  float shift[2], best[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {          // (kMaxLists)
    const bool in = lane + 32 * x < lists;
    base[x] = in ? __ldcg(&p[lane + 32 * x].base) : -INFINITY;
    sum[x] = in ? __ldcg(&p[lane + 32 * x].sum) : 0.0;
    shift[x] = in ? __ldcg(&p[lane + 32 * x].shift) : -INFINITY;
    best[x] = in ? __ldcg(&p[lane + 32 * x].best) : -INFINITY;
  }
  const float m = warp_max(fmaxf(best[0], best[1])), most = ceilf(m * kLog2e);      // (`most` is the largest shift)
  if (__any_sync(0xffffffffu, shift[0] != shift[0] || shift[1] != shift[1])) {
    const double to = fabsf(m) < kLarge ? (double)most * kLn2 : (double)m;
#pragma unroll 1
    for (int x = 0; x < 2; ++x) t += sum[x] == 0.0 ? 0.0 : sum[x] * exp(base[x] - to);
  } else {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float down = fminf(most - shift[x], 1000.0f);
      t += sum[x] * __longlong_as_double((long long)(1023 - (int)down) << 52);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  if (fabsf(m) < kLarge) t = (t - (double)exp2_fast(fmaf(m, kLog2e, -most))) * exp((double)most * kLn2 - (double)m) + 1.0;
  top = m;
  norm = log(t);
}

// The choice for an item, by the whole CTA.  A row belongs to a warp, or to as many as there are when beams are few.  Instructions, more than memory, are
// what this costs: it runs once.
template <typename T>
__device__ __noinline__ void choose(const BeamArgs& a, BeamShared& sh, int local) {
  constexpr int N = Piece<T>::N;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.beams, item = a.first_item + local;
  const BeamPart* parts = static_cast<const BeamPart*>(a.ws) + (long long)local * K * a.lists;
  const T* rows = static_cast<const T*>(a.logits) + (long long)item * K * a.ld;
  if (tid == 0) sh.count = sh.hots = 0;
  const int mates = mates_of(K), w0 = warp / mates, dw = kBeamWarps / mates;      // rows of this warp
  const int quads = a.lists * 8, q0 = (warp - w0 * mates) * 32 + lane, dq = mates * 32;                       // four lanes' maxima at a time
  auto quad = [&](int w, int q) {
    return q < quads ? __ldcg(reinterpret_cast<const float4*>(parts[w * a.lists + (q >> 3)].high) + (q & 7))
                     : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  };
  auto most_of = [](const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); };
  // The W-th largest of the lanes' maxima, and the lanes that reach it, both in fp32, as x - from + offset, and with room for its roundings:
  // `from` and `offset` are off by 2^-24 of themselves, and so are the two sums.
  float high = -INFINITY;
  float4 v[kHeld];
#pragma unroll 1
  for (int w = w0; w < K; w += dw) {
    const float score = a.scores[item * K + w];
    const bool fin = a.finished && a.finished[item * K + w];
#pragma unroll                          // on their way while the row is summed up
    for (int x = 0; x < kHeld; ++x) v[x] = quad(w, q0 + x * dq);
    double top, norm;
    sum_row(parts + w * a.lists, a.lists, top, norm);
    const int kind = !(fabsf(score) < INFINITY) ? 2 : fin ? 1 : fabs(top) < INFINITY && fabs(norm) < INFINITY ? 0 : 2;
    const float from = (float)top, offset = (float)(score - norm);
    if (lane == 0) {
      sh.score[w] = score;
      sh.top[w] = top;
      sh.norm[w] = norm;
      sh.kind[w] = kind;
      sh.fin[w] = fin;
      sh.size[w] = kind ? 0.0f : fabsf(offset) + fminf(fabsf(from), 2.0f * kLarge);
    }
    if (kind == 0) {
      float most = most_of(v[0]);
#pragma unroll
      for (int x = 1; x < kHeld; ++x) most = fmaxf(most, most_of(v[x]));
#pragma unroll 4
      for (int q = q0 + kHeld * dq; q < quads; q += dq) most = fmaxf(most, most_of(quad(w, q)));
      high = fmaxf(high, most - from + offset);
    } else if (q0 < min(K, a.vocab)) {
      high = fmaxf(high, kind == 1 && a.eos >= 0 && q0 == 0 ? score : -INFINITY);
    }
  }
  float limit = kth_largest(high, K, sh.lists);                // (its barriers cover sh)
  bool wide = limit == -INFINITY;
  if (!wide) {
    const float size = warp_max(lane < K ? sh.size[lane] : 0.0f);
    limit -= (size + fabsf(limit)) * 0x1p-21f;
#pragma unroll 1
    for (int w = w0; w < K; w += dw) {
      if (sh.kind[w]) {
        int token;
        const double total = special(a, sh, w, q0, token);
        if (q0 < min(K, a.vocab) && total >= limit) {
          const int at = atomicAdd(&sh.count, 1);
          if (at < kItemPool) {
            sh.totals[at] = total;
            sh.keys[at] = (unsigned long long)w << 32 | (unsigned)token;
            sh.orders[at] = 0;
          }
        }
        continue;
      }
      const float from = (float)sh.top[w], d = (float)((double)limit - sh.score[w] + sh.norm[w]), least = d - (size + fabsf(d)) * 0x1p-21f;
      sh.from[w] = from;
      sh.least[w] = least;
      if (high < limit) continue;                               // none of this thread's, in any row
#pragma unroll 1
      for (int q = q0; q < quads; q += kHeld * dq) {
        if (K > dw || quads > kHeld * dq) {                           // (else this thread still has them)
#pragma unroll
          for (int x = 0; x < kHeld; ++x) v[x] = quad(w, q + x * dq);
        }
        unsigned mine = 0;
#pragma unroll
        for (int x = 0; x < kHeld; ++x)            // (`least` may be -inf, which the places behind a row's maxima reach)
          if (q + x * dq < quads)
            mine |= ((v[x].x - from >= least) | (v[x].y - from >= least) << 1 | (v[x].z - from >= least) << 2 | (v[x].w - from >= least) << 3) << 4 * x;
#pragma unroll 1
        for (; mine; mine &= mine - 1) {
          const int at = atomicAdd(&sh.hots, 1), i = __ffs(mine) - 1;
          if (at < kHotLanes) sh.hot[at] = (w * quads + q + (i >> 2) * dq) * 4 + (i & 3);
        }
      }
    }
    __syncthreads();
    const int hots = sh.hots;
    if (hots <= kHotLanes) {
      // A hot lane's pieces by as many lanes as there are pieces.
      const int pieces = min(32, (min(a.chunk, a.vocab) + 32 * N - 1) / (32 * N)), width = pieces > 2 ? 1 << (31 - __clz(pieces - 1)) : 1;
#pragma unroll 1
      for (int h = tid / width; h < hots; h += kBeamThreads / width) {
        const int j = sh.hot[h], part = j >> 5, w = part / a.lists;
        const T* row = rows + w * a.ld;
        const int begin = (part - w * a.lists) * a.chunk, end = min(a.vocab, begin + a.chunk);
        const float from = sh.from[w], least = sh.least[w];
#pragma unroll 1
        for (int i0 = begin + 32 * (tid & (width - 1)) * N; i0 < end; i0 += 2 * width * 32 * N) {
          const int i1 = i0 + width * 32 * N;
          const Piece<T> p[2] = {a.vec ? load_group<T, true>(row, i0, j & 31, end) : load_group<T, false>(row, i0, j & 31, end),
                                 a.vec ? load_group<T, true>(row, i1, j & 31, end) : load_group<T, false>(row, i1, j & 31, end)};
          unsigned mine = 0;
#pragma unroll
          for (int e = 0; e < 2 * N; ++e)
            mine |= (unsigned)(p[e / N].at(e % N) - from >= least && place_in<T>(e < N ? i0 : i1, j & 31, e % N, a.vec) < end) << e;
#pragma unroll 1
          for (; mine; mine &= mine - 1) {
            const int e = __ffs(mine) - 1;
            float x = p[0].at(0);
#pragma unroll
            for (int n = 1; n < 2 * N; ++n) x = e == n ? p[n / N].at(n % N) : x;
            const int at = atomicAdd(&sh.count, 1);
            if (at < kItemPool) {
              sh.totals[at] = total_of(sh, w, x);
              sh.orders[at] = (unsigned)(rank_key(x, 0) >> 32);
              sh.keys[at] = (unsigned long long)w << 32 | (unsigned)place_in<T>(e < N ? i0 : i1, j & 31, e & (N - 1), a.vec);
            }
          }
        }
      }
    }
    __syncthreads();
    wide = sh.hots > kHotLanes || sh.count > kItemPool;
  }
  auto put = [&](int rank, double total, unsigned long long key) {
    const int w = (int)(key >> 32), tok = (int)(unsigned)key, out = item * K + rank;
    a.out_scores[out] = (float)total;
    a.out_parents[out] = item * K + w;
    a.out_tokens[out] = tok;
    a.out_finished[out] = sh.fin[w] || tok == a.eos;
  };
  if (wide) {
    __syncthreads();
    best_of_rows<T>(a, sh, rows, parts);
    if (warp > 0) return;
    // Lane w has row w's continuations, best first; the best of the lanes' next ones, K times.
    int i = 0;
#pragma unroll 1
    for (int rank = 0; rank < K; ++rank) {
      const bool in = lane < K && i < K;
      const unsigned long long mine = in ? sh.keys[lane * K + i] : ~0ull;
      unsigned long long key = mine;
      double total = in ? sh.totals[lane * K + i] : -INFINITY;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double t = __shfl_xor_sync(0xffffffffu, total, o);
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, key, o);
        if (t > total || (t == total && k < key)) {
          total = t;
          key = k;
        }
      }
      if (mine == key && key != ~0ull) {
        put(rank, total, key);
        ++i;
      }
    }
    return;
  }
  const int found = sh.count;
  for (int i = tid; i < found; i += kBeamThreads) {
    const double t = sh.totals[i];
    const unsigned long long key = sh.keys[i];
    int rank = 0, equal = 0;
    for (int j = 0; j < found; ++j) {
      rank += sh.totals[j] > t;
      equal += sh.totals[j] == t;
    }
    // Of equal totals the lower beam's; of one beam the larger logit's, which its total may be too coarse to tell; then the lower token's.
    if (equal > 1 && rank < K) {
      const unsigned order = sh.orders[i];
#pragma unroll 1
      for (int j = 0; j < found; ++j) {
        const unsigned long long other = sh.keys[j];
        const bool by_key = (other ^ key) >> 32 || sh.orders[j] == order;
        rank += sh.totals[j] == t && (by_key ? other < key : sh.orders[j] > order);
      }
    }
    if (rank < K) put(rank, t, key);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kBeamThreads, 4)
beam_kernel(const __grid_constant__ BeamArgs a) {
  constexpr int N = Piece<T>::N, U = 4;           // pieces in flight
  __shared__ BeamShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.beams;
  // An item has whole CTAs to itself.
  const int units = K * a.lists, ctas = (units + kBeamWarps - 1) / kBeamWarps, local = blockIdx.x / ctas;
  const int unit = (blockIdx.x - local * ctas) * kBeamWarps + warp, w = unit / a.lists, list = unit - w * a.lists;
  if (unit < units) {
    const T* row = static_cast<const T*>(a.logits) + ((long long)(a.first_item + local) * K + w) * a.ld;
    const int begin = list * a.chunk, end = min(a.vocab, begin + a.chunk);
    // Sums of 2^(x log2(e) - shift): `shift` is a whole number, so that sums are brought to another one exactly, and stands for shift / log2(e),
    // divided out in 64 bits, so that the rounding of log2(e) moves no sum against another.  What is left is the error of an exponential, 2^-22, and of
    // sums of 32 in 32 bits: 1e-7 of a logarithm, where a total of -20 is rounded to 1e-6.  (Exponentials in 64 bits, some 30 multiply-adds each, would
    // bound the pass by far: 33 million logits in 50 us at 18e12 of them a second, where memory takes 10.)  Maxima that are too large for it (masks of the
    // type's lowest value among them) go by differences, from themselves.
    float m = -INFINITY, shift = 0.0f;
    double s = 0.0;
    for (int i = begin; i < end; i += U * 32 * N) {
      Piece<T> p[U];
      if (VEC && i + U * 32 * N <= end) {
#pragma unroll
        for (int u = 0; u < U; ++u) p[u] = load_whole<T>(row, i + (u * 32 + lane) * N);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) p[u] = load_group<T, VEC>(row, i + u * 32 * N, lane, end);
      }
      const float top = fmaxf(fmaxf(p[0].top(), p[1].top()), fmaxf(p[2].top(), p[3].top()));
      if (top > m) {
        const float next = ceilf(top * kLog2e);
        s = rescaled(s, m, shift, top, next);
        shift = next;
        m = top;
      }
      float t[2] = {0.0f, 0.0f};
      if (fabsf(m) < kLarge) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e) t[e & 1] += exp2_fast(fmaf(p[u].at(e), kLog2e, -shift));
      } else {
        const float from = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < N; ++e) t[0] += exp2_fast((p[u].at(e) - from) * kLog2e);
      }
      s += (double)(t[0] + t[1]);
    }
    const float best = warp_max(m), last = ceilf(best * kLog2e);
    double sum = best == -INFINITY ? s : rescaled(s, m, shift, best, last);
    const double base = fabsf(best) < kLarge ? (double)last * kLn2 : (double)best;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    BeamPart* part = static_cast<BeamPart*>(a.ws) + (long long)local * units + unit;
    part->high[lane] = m;
    if (lane == 0) {
      part->sum = sum;           // NaN where there is one
      part->best = best;
      part->base = base;
      part->shift = fabsf(best) < kLarge ? last : sum == 0.0 ? -INFINITY : NAN;
    }
  }
  __syncthreads();
  if (tid == 0) {
    unsigned before;      // releases what the CTA has written (the barrier above), acquires what those before it have (the one below)
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + local) : "memory");
    sh.last = before == (unsigned)ctas - 1;
    if (sh.last) a.counters[local] = 0;
  }
  __syncthreads();
  if (sh.last) choose<T>(a, sh, local);
}

}  // namespace dptb

using namespace dptb;

extern "C" int dptb_beam_step(const BeamArgs* args, void* stream) {
  BeamArgs a = *args;
  if (a.items == 0) return 0;
  if (a.items < 0 || a.beams <= 0 || a.beams > kMaxBeams || a.vocab <= 0 || a.vocab > 1 << 30 || a.ld < 0 || (long long)a.items * a.beams > 1 << 20 ||
      (reinterpret_cast<uintptr_t>(a.ws) & 7))
    return kErrBadShape;
  // Logits of a warp: a row's share when all that are resident (32 an SM) have one, and not so many parts of a row that the choice among them is
  // what takes the time; four parts at least, so that one live beam has as many lanes to choose from as a search may have beams; a piece a lane.
  const int unit = 32 * (a.f32 ? 4 : 8), most_lists = kMaxLists;
  const long long rows = (long long)a.items * a.beams, warps = 32LL * sm_count();
  auto up = [](long long n, long long d) { return (n + d - 1) / d; };
  long long chunk = max(up((long long)a.vocab * rows, warps), 4LL * unit);
  chunk = min(chunk, up(a.vocab, 4));
  chunk = max(chunk, up(a.vocab, most_lists));
  // A little more if a row's maxima then fit the choice's registers (four rows of 50257 in fp32 9.6 us in 50 parts, 8.9 in 33); not at the price of many
  // more rounds in a row.
  const long long held = up(a.vocab, 4 * kHeld * mates_of(a.beams));
  if (a.beams <= kBeamWarps && held <= 12 * unit) chunk = max(chunk, held);
  chunk = up(chunk, chunk >= 4 * unit ? 4 * unit : unit) * (chunk >= 4 * unit ? 4 * unit : unit);
  a.chunk = (int)chunk;
  a.lists = (int)((a.vocab + chunk - 1) / chunk);
  const int size = a.f32 ? 4 : 2;
  a.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld * size % 16 == 0;
  // Items that the workspace and the counters hold go together.
  const long long part = (long long)a.beams * a.lists * (long long)sizeof(BeamPart);
  const int most = (int)min((long long)a.num_counters, a.ws_bytes / part);
  if (most < 1) return kErrTooLarge;
  auto st = static_cast<cudaStream_t>(stream);
  int launches = 0;
  for (a.first_item = 0; a.first_item < a.items; a.first_item += most, ++launches) {
    const unsigned grid = (unsigned)(min(most, a.items - a.first_item) * up((long long)a.beams * a.lists, kBeamWarps));
    auto kernel = a.f32 ? a.vec ? beam_kernel<float, true> : beam_kernel<float, false>
                        : a.vec ? beam_kernel<__nv_bfloat16, true> : beam_kernel<__nv_bfloat16, false>;
    kernel<<<grid, kBeamThreads, 0, st>>>(a);
  }
  return counted(launches, (int)cudaGetLastError());
}
