// Attention of one new token per sequence over a key / value cache in pages.
//
//   o[r, h] = sum_j softmax_j(scale * q[r, h] . k_j) v_j,   j < lens[r],
//
// where key j of row r is token j % page of page table[r, j / page], and the query heads h of a group share kv head h / G.  A row of
// length zero gives zeros.  Positions from lens[r] on are never read as numbers: what lies there may be anything.  A page number
// outside the pool hides its keys and records kBadPage in the status word, which the host turns into an exception.
//
// paged_attention_simple_kernel: a CTA per (row, query head); tiles of 128 keys, a thread a key for the scores and a thread a feature for
// the weighted sum; fp32 throughout.
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
};

constexpr int kSimpleTile = 128;
constexpr int kMaxHeadDim = 256;

template <typename T>
__global__ void __launch_bounds__(kSimpleTile)
paged_attention_simple_kernel(const PagedAttnArgs a) {
  __shared__ float s_q[kMaxHeadDim], s_p[kSimpleTile], s_red[33];
  __shared__ int s_page[kSimpleTile];
  const int h = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  const int g = h / (a.heads / a.kv_heads);
  const int room = (int)min((long long)a.width * a.page, 0x7fffffffLL);
  int n = a.lens[r];
  if (n > room) {
    if (tid == 0) report_error(kBadPage);
    n = room;
  }
  const T* q = static_cast<const T*>(a.q) + r * a.q_row + h * a.q_head;
  for (int d = tid; d < a.hd; d += kSimpleTile) s_q[d] = to_f32(q[d]) * a.scale;
  const T* kb = static_cast<const T*>(a.k) + g * a.k_head;
  const T* vb = static_cast<const T*>(a.v) + g * a.v_head;
  float m = -INFINITY, l = 0.0f, acc[kMaxHeadDim / kSimpleTile] = {};
  for (int j0 = 0; j0 < n; j0 += kSimpleTile) {
    const int j = j0 + tid, nt = min(kSimpleTile, n - j0);
    int page = -1;
    if (j < n) {
      page = a.table[r * a.table_row + j / a.page];
      if (page < 0 || page >= a.pages) {
        report_error(kBadPage);
        page = -1;
      }
    }
    __syncthreads();
    s_page[tid] = page;
    __syncthreads();
    float s = -INFINITY;
    if (page >= 0) {
      const T* k = kb + page * a.k_page + (j % a.page) * a.k_tok;
      s = 0.0f;
      for (int d = 0; d < a.hd; ++d) s += s_q[d] * to_f32(k[d]);
    }
    const float nm = fmaxf(m, block_max(s, s_red)), sub = nm == -INFINITY ? 0.0f : nm;
    const float corr = __expf(m - sub), p = page >= 0 ? __expf(s - sub) : 0.0f;
    l = l * corr + block_sum(p, s_red);
    m = nm;
    s_p[tid] = p;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / kSimpleTile; ++i) {
      const int d = i * kSimpleTile + tid;
      if (d >= a.hd) break;
      float t = acc[i] * corr;
      for (int x = 0; x < nt; ++x) {
        const int pg = s_page[x];
        if (pg >= 0) t += s_p[x] * to_f32(vb[pg * a.v_page + ((j0 + x) % a.page) * a.v_tok + d]);
      }
      acc[i] = t;
    }
  }
  T* o = static_cast<T*>(a.o) + r * a.o_row + h * a.o_head;
#pragma unroll
  for (int i = 0; i < kMaxHeadDim / kSimpleTile; ++i) {
    const int d = i * kSimpleTile + tid;
    if (d < a.hd) o[d] = from_f32<T>(n > 0 ? acc[i] / l : 0.0f);
  }
}

}  // namespace dptb

using namespace dptb;

extern "C" int dptb_paged_attention(const PagedAttnArgs* args, void* stream) {
  const PagedAttnArgs& a = *args;
  if (a.rows == 0 || a.heads == 0) return 0;
  if (a.rows < 0 || a.rows > 65535 || a.heads < 0 || a.kv_heads <= 0 || a.heads % a.kv_heads || a.hd <= 0 || a.hd > kMaxHeadDim ||
      a.page <= 0 || a.width < 0 || a.pages < 0)
    return kErrBadShape;
  const dim3 grid(a.heads, a.rows);
  auto st = static_cast<cudaStream_t>(stream);
  if (a.f32) paged_attention_simple_kernel<float><<<grid, kSimpleTile, 0, st>>>(a);
  else       paged_attention_simple_kernel<__nv_bfloat16><<<grid, kSimpleTile, 0, st>>>(a);
  return counted(1, (int)cudaGetLastError());
}
