// Attention of a chunk of new tokens over the paged cache: query row (token t
// of request b, head h) at position p = length_b - n_b + i (i: the token's
// place among the request's n_b) sees the keys lo <= j < hi,
//   hi = max(p + 1, prefix_b), lo = max(0, p + 1 - window, key_start_t),
// with scores x_j = scale q.k_j, capped to softcap tanh(x_j / softcap), less
// slope_h |p - j|; the output is sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),
// zeros where no key is seen.
#pragma once

#include <cuda_bf16.h>

#include "bc_attn.cuh"

namespace bc {

struct ChunkParams {
  int batch, tokens, hq, hkv, group;
  int max_pages, physical_pages;
  int window;                 // 0: none
  const void* q;
  long long q_stride;         // elements between two tokens' rows
  const void* k;
  const void* v;
  long long block_stride, slot_stride, head_stride;  // elements
  const int* pages;           // [batch, max_pages]
  const int* query_start;     // [batch + 1]
  const int* lengths;         // [batch]
  const int* prefix;          // [batch] or null
  const int* key_start;       // [tokens] or null
  const float* slopes;        // [hq] or null
  void* out;                  // [tokens, hq, D]
  int out_f32;
  float scale, softcap;       // softcap 0: none
  unsigned* err;
  unsigned token;
};

// A request's rows and keys, with malformed values brought into range.
struct ChunkRequest {
  int first, n, len;  // first token, tokens, keys
};
__device__ __forceinline__ ChunkRequest chunk_request(const ChunkParams& p, int b) {
  const int a = p.query_start[b], e = p.query_start[b + 1], len = p.lengths[b];
  ChunkRequest r;
  r.first = min(max(a, 0), p.tokens);
  r.n = max(min(e, p.tokens) - r.first, 0);
  r.len = min(max(len, 0), p.max_pages * kPageSize);
  if (a != r.first || e != r.first + r.n || len != r.len || r.len < r.n) atomicOr(p.err, kErrLength);
  return r;
}

// A warp per query row: every lane takes a key at a time, then a share of the
// output's dimensions.
template <int D, typename T>
__global__ void __launch_bounds__(128) chunk_rows_kernel(const ChunkParams p) {
  __shared__ float s_q[4][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  const long long row = (long long)blockIdx.x * 4 + warp;
  if (row >= (long long)p.tokens * p.hq) return;
  const int t = int(row / p.hq), h = int(row % p.hq);
  int lo = 0, hi = p.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.query_start[mid] <= t) lo = mid; else hi = mid;
  }
  const ChunkRequest rq = chunk_request(p, lo);
  if (t < rq.first || t >= rq.first + rq.n) return;
  const int pos = rq.len - rq.n + (t - rq.first);
  int end = pos + 1, begin = 0;
  if (p.prefix) end = max(end, min(p.prefix[lo], rq.len));
  if (p.window) begin = max(begin, pos + 1 - p.window);
  if (p.key_start) begin = max(begin, p.key_start[t]);
  const T* q = static_cast<const T*>(p.q) + t * p.q_stride + size_t(h) * D;
  for (int d = lane; d < D; d += 32) s_q[warp][d] = float(q[d]);
  __syncwarp();
  const int kvh = h / p.group;
  const float slope = p.slopes ? p.slopes[h] : 0.f;
  float m = -INFINITY, l = 0.f, acc[D / 32];
#pragma unroll
  for (int r = 0; r < D / 32; ++r) acc[r] = 0.f;
  for (int j0 = begin; j0 < end; j0 += 32) {
    const int j = j0 + lane;
    float x = -INFINITY;
    long long at = -1;
    if (j < end) {
      const int page = p.pages[size_t(lo) * p.max_pages + j / kPageSize];
      x = 0.f;
      if (page < 0 || page >= p.physical_pages) {
        atomicOr(p.err, kErrPageRange);
      } else {
        at = page * p.block_stride + (j % kPageSize) * p.slot_stride + kvh * p.head_stride;
        for (int d = 0; d < D; ++d) x += s_q[warp][d] * float(static_cast<const T*>(p.k)[at + d]);
      }
      x *= p.scale;
      if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
      x -= slope * fabsf(float(pos - j));
    }
    float mx = x;
    for (int d = 1; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float mn = fmaxf(m, mx), a = expf(m - mn), w = expf(x - mn);
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int r = 0; r < D / 32; ++r) acc[r] *= a;
    for (int k = 0; k < min(32, end - j0); ++k) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      const long long ak = __shfl_sync(0xffffffffu, at, k);
      if (ak < 0) continue;
#pragma unroll
      for (int r = 0; r < D / 32; ++r)
        acc[r] += wk * float(static_cast<const T*>(p.v)[ak + r * 32 + lane]);
    }
  }
  for (int d = 1; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int r = 0; r < D / 32; ++r) {
    const size_t o = size_t(row) * D + r * 32 + lane;
    if (p.out_f32)
      static_cast<float*>(p.out)[o] = acc[r] * inv;
    else
      static_cast<T*>(p.out)[o] = T(acc[r] * inv);
  }
}

}  // namespace bc
