// Beam search's selection: of all continuations of an item's beams, the best as many as it has beams.
//
//   total[b, w, v] = score[b, w] + logit[b * W + w, v] - log sum_u exp(logit[b * W + w, u])
//
// Candidates are ranked by (total, then the lower w * V + v).  A finished beam has one continuation, `eos` at its old score; its others, those
// of a beam whose score is -inf or NaN, and those of a row of logits without a distribution (a NaN, an infinity, nothing but
// -inf) are worth -inf.  Within a beam the order is that of the logits themselves, so that no rounding decides it; totals of different beams
// meet in 64 bits.
//
// beam_rows_kernel: a CTA per row of logits; its maximum and sum of exponentials, and its best W by as many passes.
// beam_merge_kernel: a warp per item; lane w holds beam w's sorted list, and W times the best head of the lists is taken.
#include <cuda_bf16.h>

#include "common/host.h"
#include "common/reduce.cuh"

namespace dptb {

constexpr int kMaxBeams = 32;
constexpr int kBeamThreads = 512;

struct BeamArgs {
  const void* logits;            // [items * beams, ld]
  const float* scores;           // [items, beams]
  const unsigned char* finished; // [items, beams] or null
  float* out_scores;
  int* out_parents;              // row of the parent
  long long* out_tokens;
  unsigned char* out_finished;
  void* ws;
  long long ld, ws_bytes;
  int items, beams, vocab, eos, f32;
};
static_assert(sizeof(BeamArgs) == 104, "packed by the caller");

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

template <typename T>
__global__ void __launch_bounds__(kBeamThreads)
beam_rows_kernel(const BeamArgs a, unsigned long long* best, double* norm) {
  __shared__ float red[33];
  __shared__ double dsum[kBeamThreads / 32];
  __shared__ unsigned long long kred[kBeamThreads / 32];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* x = static_cast<const T*>(a.logits) + r * a.ld;
  float m = -INFINITY;
  for (int v = tid; v < a.vocab; v += kBeamThreads) m = fmaxf(m, to_f32(x[v]));
  m = block_max(m, red);
  double s = 0.0;
  for (int v = tid; v < a.vocab; v += kBeamThreads) s += expf(to_f32(x[v]) - m);
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) dsum[warp] = s;
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < kBeamThreads / 32; ++w) t += dsum[w];
    norm[2 * r] = m;
    norm[2 * r + 1] = log(t);      // NaN where the row has no distribution
  }
  unsigned long long last = ~0ull;
  for (int i = 0; i < min(a.beams, a.vocab); ++i) {
    unsigned long long top = 0;
    for (int v = tid; v < a.vocab; v += kBeamThreads) {
      const unsigned long long k = rank_key(to_f32(x[v]), v);
      if (k < last && k > top) top = k;
    }
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    __syncthreads();
    if (lane == 0) kred[warp] = top;
    __syncthreads();
    for (int w = 0; w < kBeamThreads / 32; ++w) top = max(top, kred[w]);
    if (tid == 0) best[(long long)r * a.beams + i] = top;
    last = top;
  }
}

__global__ void __launch_bounds__(32)
beam_merge_kernel(const BeamArgs a, const unsigned long long* best, const double* norm) {
  const int b = blockIdx.x, w = threadIdx.x, W = a.beams;
  const int row = b * W + w, count = min(W, a.vocab);
  const double kNone = -INFINITY;
  double score = kNone, top = 0.0, z = 0.0;
  bool fin = false, dead = true;
  if (w < W) {
    score = a.scores[row];
    fin = a.finished && a.finished[row];
    top = norm[2 * row];
    z = norm[2 * row + 1];
    dead = !(score > kNone) || !(fabs(z) < INFINITY);
    if (fin && score > kNone) dead = false;
  }
  int at = 0, token = 0;
  double total = kNone;
  auto head = [&] {      // entry `at` of this beam's list, best first
    if (w >= W) return;
    if (dead) {
      token = at;
    } else if (fin) {
      const bool has = a.eos >= 0 && a.eos < a.vocab;
      if (has && at == 0) {
        token = a.eos;
        total = score;
      } else {
        token = at - has;
        if (has && token >= a.eos) ++token;
        total = kNone;
      }
    } else {
      const unsigned long long k = best[(long long)row * W + at];
      token = key_index(k);
      total = score + ((double)key_value(k) - top - z);     // (a row masked by the lowest value loses nothing to its size)
      if (total != total) total = kNone;      // an infinite score on a token of no probability
    }
  };
  head();
  for (int i = 0; i < W; ++i) {
    double t = total;
    int who = w < W && at < count ? w : 64;     // lists that are used up come last
    for (int o = 16; o > 0; o >>= 1) {
      const double u = __shfl_xor_sync(0xffffffffu, t, o);
      const int x = __shfl_xor_sync(0xffffffffu, who, o);
      if (x < 64 && (who == 64 || u > t || (u == t && x < who))) {
        t = u;
        who = x;
      }
    }
    if (w == who) {
      const int out = b * W + i;
      a.out_scores[out] = (float)total;
      a.out_parents[out] = row;
      a.out_tokens[out] = token;
      a.out_finished[out] = fin || token == a.eos;
      if (++at < count) head();
    }
  }
}

}  // namespace dptb

using namespace dptb;

extern "C" long long dptb_beam_ws_bytes(int items, int beams) { return (long long)items * beams * (beams + 2) * 8; }

extern "C" int dptb_beam_step(const BeamArgs* args, void* stream) {
  const BeamArgs& a = *args;
  if (a.items == 0) return 0;
  if (a.items < 0 || a.beams <= 0 || a.beams > kMaxBeams || a.vocab <= 0 || a.ld < 0 || (long long)a.items * a.beams > 1 << 20 ||
      (reinterpret_cast<uintptr_t>(a.ws) & 7))
    return kErrBadShape;
  if (a.ws_bytes < dptb_beam_ws_bytes(a.items, a.beams)) return kErrTooLarge;
  const int rows = a.items * a.beams;
  auto st = static_cast<cudaStream_t>(stream);
  auto* best = static_cast<unsigned long long*>(a.ws);
  auto* norm = reinterpret_cast<double*>(best + (long long)rows * a.beams);
  if (a.f32) beam_rows_kernel<float><<<rows, kBeamThreads, 0, st>>>(a, best, norm);
  else       beam_rows_kernel<__nv_bfloat16><<<rows, kBeamThreads, 0, st>>>(a, best, norm);
  beam_merge_kernel<<<a.items, 32, 0, st>>>(a, best, norm);
  return counted(2, (int)cudaGetLastError());
}
