// Beam search's selection: of all continuations of an item's beams, the best as many as it has beams.
//
//   total[b, w, v] = score[b, w] + logit[b * W + w, v] - log sum_u exp(logit[b * W + w, u])
//
// Candidates are ranked by (total, then the lower w * V + v).  A finished beam has one continuation, `eos` at its old score; its others, those
// of a beam whose score is -inf or NaN, and those of a row of logits without a distribution (a NaN, an infinity, nothing but
// -inf) are worth -inf.  Within a beam the order is that of the logits themselves, so that no rounding decides it; totals of different beams
// meet in 64 bits.
//
// beam_kernel: a row is dealt to a few CTAs (chunks).  One pass over the logits keeps a running maximum and sum of exponentials in every
// thread; that is all that is done for each logit.  The best W of a chunk lie with the threads of the W largest maxima, so those alone look at
// their logits again and hand in what is not below the W-th of these maxima: W values and a few more, whatever the vocabulary.  The
// last CTA of an item (a counter, no waiting) sums up its rows and chooses among their lists in the same way.
//
// Bound by memory for many rows, by a chain of latencies for few.
#include <cuda_bf16.h>

#include "common/host.h"
#include "common/reduce.cuh"

namespace dptb {

constexpr int kMaxBeams = 32;
constexpr int kBeamThreads = 512, kBeamWarps = kBeamThreads / 32;
constexpr int kBeamPool = 1024;        // candidates that are ranked at once
constexpr int kMaxChunks = 32;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamArgs {
  const void* logits;            // [items * beams, ld]
  const float* scores;           // [items, beams]
  const unsigned char* finished; // [items, beams] or null
  float* out_scores;
  int* out_parents;              // row of the parent
  long long* out_tokens;
  unsigned char* out_finished;
  void* ws;                      // per row and chunk: sum of exponentials, maximum, the best keys
  unsigned* counters;            // a zeroed word per item of a launch; zero again afterwards
  long long ld, ws_bytes;
  int items, beams, vocab, eos, f32, num_counters;
  int chunk, chunks, vec, first_item;   // set by the launcher
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

// The k-th largest of the block's values, k <= 32: warps sort theirs, and lists are merged pairwise, the 32 largest of two at a time.
__device__ __forceinline__ float kth_largest(float v, int k, float* lists) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1)
#pragma unroll
    for (int j = n >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, j);
      v = ((lane & j) == 0) == ((lane & n) == 0) ? fmaxf(v, o) : fminf(v, o);
    }
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

// A thread's pieces of a row: 16 bytes each, kBeamThreads pieces apart.
template <typename T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  T e[N];
  // Elements first .. first + N of a row of `end`; those beyond are -inf.
  __device__ __forceinline__ void load(const T* row, int first, int end, bool vec) {
    if (vec && first + N <= end) {
      *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(row + first);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = first + i < end ? row[first + i] : from_f32<T>(-INFINITY);
    }
  }
};

struct BeamShared {
  float lists[kBeamThreads];
  float red[33];
  double sums[kBeamWarps];
  unsigned long long keys[kBeamPool];      // of a chunk; of the item: (beam, token)
  double totals[kBeamPool];
  double score[kMaxBeams], top[kMaxBeams], norm[kMaxBeams];
  unsigned char kind[kMaxBeams];           // 0: by its logits, 1: finished, 2: nothing to offer
  int count, scan[33], last;
};

__device__ __forceinline__ int block_scan_total(int v, int* scratch, int& total) {      // exclusive sum
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
  int before = 0;
  total = 0;
  for (int w = 0; w < kBeamWarps; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  return before + s - v;
}

// Of the logits [begin, end) the best `count` as keys in `out`, best first, 0 behind the last.  Threads hand in what is not below the threshold; where too many
// logits equal it (a masked vocabulary), those above it, and the first of the equal ones in their order.
template <typename T>
__device__ __forceinline__ void best_of_chunk(const BeamArgs& a, const T* row, int begin, int end, float mine, unsigned long long* out, BeamShared& sh) {
  constexpr int N = Piece<T>::N;
  const int tid = threadIdx.x, K = a.beams;
  const float limit = kth_largest(mine, K, sh.lists);
#pragma unroll 1
  for (int round = 0; round < 2; ++round) {
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (round == 0 ? mine >= limit : mine > limit) {
#pragma unroll 4
      for (int i = begin + tid * N; i < end; i += kBeamThreads * N) {
        Piece<T> p;
        p.load(row, i, end, a.vec);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float x = to_f32(p.e[e]);
          if (i + e < end && (round == 0 ? x >= limit : x > limit)) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kBeamPool) sh.keys[at] = rank_key(x, i + e);
          }
        }
      }
    }
    __syncthreads();
    const int above = sh.count;                   // (everybody's, before it changes)
    __syncthreads();
    if (above <= kBeamPool - (round ? K : 0)) {
      if (round == 0) break;
      int found = above;
      for (int i0 = begin; i0 < end && found - above < K; i0 += kBeamThreads * N) {
        const int i = i0 + tid * N;
        Piece<T> p;
        p.load(row, i, end, a.vec);
        int equal = 0, total;
#pragma unroll
        for (int e = 0; e < N; ++e) equal += i + e < end && to_f32(p.e[e]) == limit;
        int at = found + block_scan_total(equal, sh.scan, total);
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (i + e < end && to_f32(p.e[e]) == limit) {
            if (at - above < K) sh.keys[at] = rank_key(limit, i + e);
            ++at;
          }
        found += total;
      }
      __syncthreads();
      if (tid == 0) sh.count = min(found, above + K);
      __syncthreads();
      break;
    }
    if (round == 1) {
      // Too many above it as well: the best, one after the other.
      unsigned long long last = ~0ull;
      for (int k = 0; k < K; ++k) {
        unsigned long long top = 0;
        for (int i = begin + tid; i < end; i += kBeamThreads) {
          const unsigned long long key = rank_key(to_f32(row[i]), i);
          if (key < last && key > top) top = key;
        }
        for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((tid & 31) == 0) sh.keys[K + (tid >> 5)] = top;
        __syncthreads();
        for (int w = 0; w < kBeamWarps; ++w) top = max(top, sh.keys[K + w]);
        if (tid == 0) sh.keys[k] = top;
        last = top;
        __syncthreads();
      }
      if (tid == 0) sh.count = min(K, end - begin);
      __syncthreads();
    }
  }
  const int n = sh.count;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long key = sh.keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.keys[j] > key;
    if (rank < K) out[rank] = key;
  }
  for (int i = n + tid; i < K; i += kBeamThreads) out[i] = 0;
}

// Candidate c of an item: entry c % (chunks * beams) of beam c / (chunks * beams); false if there is none.
__device__ __forceinline__ bool candidate(const BeamArgs& a, const BeamShared& sh, const unsigned char* parts, long long part, int c, int& beam, int& token, double& total) {
  const int each = a.chunks * a.beams;
  beam = c / each;
  const int i = c - beam * each;
  total = -INFINITY;
  if (sh.kind[beam]) {
    if (i >= min(a.beams, a.vocab)) return false;
    token = i;
    if (sh.kind[beam] == 1 && a.eos >= 0) {       // eos first, then the others
      if (i == 0) {
        token = a.eos;
        total = sh.score[beam];
      } else {
        token = i - 1 + (i - 1 >= a.eos);
      }
    }
    return true;
  }
  const int chunk = i / a.beams;
  const unsigned long long key = __ldcg(reinterpret_cast<const unsigned long long*>(parts + (beam * (long long)a.chunks + chunk) * part + 16) + (i - chunk * a.beams));
  if (key == 0) return false;
  token = key_index(key);
  total = sh.score[beam] + ((double)key_value(key) - sh.top[beam] - sh.norm[beam]);     // (a row masked by the lowest value loses nothing to its size)
  if (total != total) total = -INFINITY;          // an infinite score on a token of no probability
  return true;
}

template <typename T>
__global__ void __launch_bounds__(kBeamThreads)
beam_kernel(const BeamArgs a) {
  constexpr int N = Piece<T>::N, U = 4;           // pieces in flight
  __shared__ BeamShared sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.beams;
  const int local = blockIdx.y / K, item = a.first_item + local;
  const int row_index = item * K + blockIdx.y % K, chunk = blockIdx.x;
  const T* row = static_cast<const T*>(a.logits) + row_index * a.ld;
  const int begin = chunk * a.chunk, end = min(a.vocab, begin + a.chunk);
  const long long part = 16 + 8LL * K;
  unsigned char* parts = static_cast<unsigned char*>(a.ws) + (long long)local * K * a.chunks * part;     // of the item
  float m = -INFINITY, s = 0.0f;
  for (int i = begin + tid * N; i < end; i += U * kBeamThreads * N) {
    Piece<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) p[u].load(row, i + u * kBeamThreads * N, end, a.vec);
    float top = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, to_f32(p[u].e[e]));
    const float base = top == -INFINITY ? 0.0f : top;
    if (top != m) s *= exp2_fast((m - base) * kLog2e);
    m = top;
    float t[2] = {0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) t[e & 1] += exp2_fast((to_f32(p[u].e[e]) - base) * kLog2e);
    s += t[0] + t[1];
  }
  const float best = block_max(m, sh.red), base = best == -INFINITY ? 0.0f : best;
  double sum = (double)(s * exp2_fast((m - base) * kLog2e));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sh.sums[warp] = sum;
  unsigned char* mine = parts + ((blockIdx.y % K) * (long long)a.chunks + chunk) * part;
  best_of_chunk<T>(a, row, begin, end, m, reinterpret_cast<unsigned long long*>(mine + 16), sh);
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < kBeamWarps; ++w) t += sh.sums[w];
    *reinterpret_cast<double*>(mine) = t;          // NaN where the chunk holds a NaN or an infinity
    *reinterpret_cast<double*>(mine + 8) = best;
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    const bool last = atomicAdd(a.counters + local, 1u) == (unsigned)(K * a.chunks) - 1;
    if (last) a.counters[local] = 0;
    sh.last = last;
    sh.count = 0;
  }
  __syncthreads();
  if (!sh.last) return;
  __threadfence();
  for (int w = warp; w < K; w += kBeamWarps) {
    const unsigned char* p = parts + (w * (long long)a.chunks + lane) * part;
    const bool in = lane < a.chunks;
    const double m_part = in ? __ldcg(reinterpret_cast<const double*>(p + 8)) : -INFINITY;
    const double s_part = in ? __ldcg(reinterpret_cast<const double*>(p)) : 0.0;
    double top = m_part;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    double t = in ? s_part * exp(m_part - (top == -INFINITY ? 0.0 : top)) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (lane == 0) {
      const float score = a.scores[item * K + w];
      const bool fin = a.finished && a.finished[item * K + w];
      const double norm = log(t);
      sh.score[w] = score;
      sh.top[w] = top;
      sh.norm[w] = norm;
      sh.kind[w] = !(score > -INFINITY) ? 2 : fin ? 1 : fabs(top) < INFINITY && fabs(norm) < INFINITY ? 0 : 2;
    }
  }
  __syncthreads();
  const int n = K * K * a.chunks;
  int beam, token;
  double total;
  float high = -INFINITY;
  for (int c = tid; c < n; c += kBeamThreads)
    if (candidate(a, sh, parts, part, c, beam, token, total)) high = fmaxf(high, (float)total);
  const float limit = kth_largest(high, K, sh.lists);          // (rounding to fp32 keeps the order)
  for (int c = tid; c < n; c += kBeamThreads)
    if (candidate(a, sh, parts, part, c, beam, token, total) && (float)total >= limit) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kBeamPool) {
        sh.totals[at] = total;
        sh.keys[at] = (unsigned long long)beam << 32 | (unsigned)token;
      }
    }
  __syncthreads();
  auto write = [&](int at, unsigned long long key, double t) {
    const int w = (int)(key >> 32), tok = (int)(unsigned)key, out = item * K + at;
    a.out_scores[out] = (float)t;
    a.out_parents[out] = item * K + w;
    a.out_tokens[out] = tok;
    a.out_finished[out] = (a.finished && a.finished[item * K + w]) || tok == a.eos;
  };
  const int found = sh.count;
  if (found <= kBeamPool) {
    for (int i = tid; i < found; i += kBeamThreads) {
      const double t = sh.totals[i];
      const unsigned long long key = sh.keys[i];
      int rank = 0;
      for (int j = 0; j < found; ++j) rank += sh.totals[j] > t || (sh.totals[j] == t && sh.keys[j] < key);
      if (rank < K) write(rank, key, t);
    }
    return;
  }
  // Too many equal ones: one after the other.
  double last_total = INFINITY;
  unsigned long long last_key = 0;
  for (int k = 0; k < K; ++k) {
    double t = -INFINITY;
    unsigned long long key = ~0ull;
    for (int c = tid; c < n; c += kBeamThreads)
      if (candidate(a, sh, parts, part, c, beam, token, total)) {
        const unsigned long long id = (unsigned long long)beam << 32 | (unsigned)token;
        const bool after = k == 0 || total < last_total || (total == last_total && id > last_key);
        if (after && (total > t || (total == t && id < key))) {
          t = total;
          key = id;
        }
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double u = __shfl_xor_sync(0xffffffffu, t, o);
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, key, o);
      if (u > t || (u == t && x < key)) {
        t = u;
        key = x;
      }
    }
    __syncthreads();
    if (lane == 0) {
      sh.totals[warp] = t;
      sh.keys[warp] = key;
    }
    __syncthreads();
    for (int w = 0; w < kBeamWarps; ++w)
      if (sh.totals[w] > t || (sh.totals[w] == t && sh.keys[w] < key)) {
        t = sh.totals[w];
        key = sh.keys[w];
      }
    if (tid == 0) write(k, key, t);
    last_total = t;
    last_key = key;
  }
}

}  // namespace dptb

using namespace dptb;

extern "C" int dptb_beam_step(const BeamArgs* args, void* stream) {
  BeamArgs a = *args;
  if (a.items == 0) return 0;
  if (a.items < 0 || a.beams <= 0 || a.beams > kMaxBeams || a.vocab <= 0 || a.vocab > 1 << 30 || a.ld < 0 || (long long)a.items * a.beams > 1 << 20 ||
      (reinterpret_cast<uintptr_t>(a.ws) & 7))
    return kErrBadShape;
  // Chunks: as many CTAs as are resident at once (4 an SM), as far as each has a round of loads to do (4 pieces a thread).
  const int rows = a.items * a.beams, unit = kBeamThreads * (a.f32 ? 4 : 8);
  long long chunk = ((long long)a.vocab * rows + 4LL * sm_count() - 1) / (4LL * sm_count());
  chunk = max(chunk, (long long)unit);
  chunk = max(chunk, ((long long)a.vocab + kMaxChunks - 1) / kMaxChunks);
  chunk = (chunk + unit - 1) / unit * unit;
  a.chunk = (int)min(chunk, 0x7fffffffLL / unit * unit);
  a.chunks = (a.vocab + a.chunk - 1) / a.chunk;
  const int size = a.f32 ? 4 : 2;
  a.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld * size % 16 == 0;
  // Items that the workspace and the counters hold go together.
  const long long part = (long long)a.beams * a.chunks * (16 + 8LL * a.beams);
  const int most = (int)min(min((long long)a.num_counters, a.ws_bytes / part), 65535LL / a.beams);
  if (most < 1) return kErrTooLarge;
  auto st = static_cast<cudaStream_t>(stream);
  int launches = 0;
  for (a.first_item = 0; a.first_item < a.items; a.first_item += most, ++launches) {
    const dim3 grid(a.chunks, min(most, a.items - a.first_item) * a.beams);
    if (a.f32) beam_kernel<float><<<grid, kBeamThreads, 0, st>>>(a);
    else       beam_kernel<__nv_bfloat16><<<grid, kBeamThreads, 0, st>>>(a);
  }
  return counted(launches, (int)cudaGetLastError());
}
