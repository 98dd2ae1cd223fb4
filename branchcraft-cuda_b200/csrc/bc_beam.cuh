// Beam search on the device: the k best (beam, token) pairs of every request
// (beam_chunk_kernel, beam_merge_kernel) and the page tables and reference
// counts after the beams' new parents (beam_rows_kernel, beam_release_kernel).
#pragma once

#include <cuda_bf16.h>

#include "bc_attn.cuh"

namespace bc {

constexpr int kBeamMax = 64;      // beams of a request
constexpr int kBeamMaxK = 64;     // pairs selected
constexpr int kBeamMaxVocab = 1 << 20;
constexpr int kBeamThreads = 512;
constexpr int kBeamPerThread = 32;
constexpr int kBeamChunk = kBeamThreads * kBeamPerThread;  // logits of one block
constexpr int kBeamGroups = kBeamThreads / 4;              // four threads each

enum BeamType : int { kBeamF16 = 0, kBeamBF16 = 1, kBeamF32 = 2 };

// A logit as the search sees it: NaN counts as -inf (never chosen before a
// number), +inf as the largest number; -0 as +0, so that equal logits are
// equal keys.
__device__ __forceinline__ float beam_logit(float x) {
  if (!(x > -INFINITY)) return -INFINITY;
  return fminf(x, 3.402823466e38f) + 0.f;
}

// Keys: larger value first, then the lower index. Unique, so selection never
// meets a tie.
__device__ __forceinline__ unsigned beam_order(float x) {
  const unsigned u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float beam_value(unsigned u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ unsigned long long beam_key(float x, unsigned index) {
  return ((unsigned long long)beam_order(x) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ unsigned long long beam_order64(double x) {
  const unsigned long long u = __double_as_longlong(x);
  return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double beam_value64(unsigned long long u) {
  return __longlong_as_double(u >> 63 ? u & ~(1ull << 63) : ~u);
}

struct BeamSelectParams {
  int batch, beams, vocab, k, chunks;
  const void* logits;
  long long row_stride;  // elements between two beams' rows
  const float* scores;   // [batch, beams]
  float* out_scores;     // [batch, k]
  int* out_tokens;
  int* out_parents;
  // workspace, per (row, chunk): the k best keys in order (0 past the
  // chunk's logits), the largest logit and the sum of exp(x - largest)
  unsigned long long* keys;  // [rows, chunks, k]
  float* chunk_max;          // [rows, chunks]
  double* chunk_sum;         // [rows, chunks]
};

// One block per chunk of a row. Every thread keeps its logits in registers;
// the threshold is the k-th largest of the 128 groups' maxima, so the chunk's
// k best lie in k groups and a few more than k logits pass it.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads) beam_chunk_kernel(const BeamSelectParams p) {
  __shared__ unsigned long long s_group[kBeamGroups];
  extern __shared__ unsigned long long s_cand[];  // [k * 4 * kBeamPerThread]
  __shared__ float s_max[kBeamThreads / 32];
  __shared__ double s_sum[kBeamThreads / 32];
  __shared__ unsigned long long s_tau;
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int first = chunk * kBeamChunk, count = min(kBeamChunk, p.vocab - first);
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride + first;
  float v[kBeamPerThread];
#pragma unroll
  for (int j = 0; j < kBeamPerThread; ++j) {
    const int i = j * kBeamThreads + tid;
    v[j] = i < count ? beam_logit(float(x[i])) : -INFINITY;
  }
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < kBeamPerThread; ++j) mx = fmaxf(mx, v[j]);
  // the largest key of the thread: its first logit equal to mx
  unsigned long long best = 0;
#pragma unroll
  for (int j = kBeamPerThread - 1; j >= 0; --j)
    if (j * kBeamThreads + tid < count && v[j] == mx) best = beam_key(mx, j * kBeamThreads + tid);
  unsigned long long g = best;
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, g, d);
    g = o > g ? o : g;
  }
  if ((lane & 3) == 0) s_group[tid >> 2] = g;
  float wm = mx;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, d));
  if (lane == 0) s_max[warp] = wm;
  if (tid == 0) {
    s_n = 0;
    s_tau = 0;
  }
  __syncthreads();
  float m = s_max[0];
#pragma unroll
  for (int w = 1; w < kBeamThreads / 32; ++w) m = fmaxf(m, s_max[w]);
  // the k-th largest group maximum (empty groups are 0 and tie below it)
  if (tid < kBeamGroups) {
    const unsigned long long mine = s_group[tid];
    int above = 0;
    for (int i = 0; i < kBeamGroups; ++i) above += s_group[i] > mine;
    if (above == p.k - 1 && mine != 0) s_tau = mine;
  }
  // the sum: expf is within 2 units in the last place; sums beyond a thread's
  // 32 terms are held in 64 bits, since the order of two beams' candidates
  // hangs on the last digits
  float part = 0.f;
  const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int j = 0; j < kBeamPerThread; ++j) part += expf(v[j] - base);
  double sum = part;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  const unsigned long long tau = s_tau;
  if (best >= tau && best != 0) {
#pragma unroll
    for (int j = 0; j < kBeamPerThread; ++j) {
      const int i = j * kBeamThreads + tid;
      if (i < count) {
        const unsigned long long key = beam_key(v[j], i);
        if (key >= tau) s_cand[atomicAdd(&s_n, 1)] = key;
      }
    }
  }
  __syncthreads();
  const int n = s_n;
  const size_t at = size_t(blockIdx.x) * p.k;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long mine = s_cand[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += s_cand[j] > mine;
    // (the index within the chunk becomes the token)
    if (above < p.k) p.keys[at + above] = mine - unsigned(first);
  }
  for (int i = n + tid; i < p.k; i += kBeamThreads) p.keys[at + i] = 0;
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < kBeamThreads / 32; ++w) s += s_sum[w];
    p.chunk_max[blockIdx.x] = m;
    p.chunk_sum[blockIdx.x] = s;
  }
}

// One block per request: the rows' log sums, then the k best of all chunks'
// lists. Lists are sorted, so the k best lie in the k lists with the best
// heads: at most k*k candidates.
__global__ void __launch_bounds__(kBeamThreads) beam_merge_kernel(const BeamSelectParams p) {
  extern __shared__ unsigned long long beam_smem[];
  __shared__ double s_off[kBeamMax];
  __shared__ float s_top[kBeamMax];
  __shared__ int s_n;
  __shared__ unsigned long long s_tau_v;
  __shared__ unsigned s_tau_i;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lists = p.beams * p.chunks;
  unsigned long long* head_v = beam_smem;                   // [lists] order of the head's score
  unsigned* head_i = reinterpret_cast<unsigned*>(head_v + lists);  // [lists] its beam*vocab + token
  unsigned long long* cand_v = head_v + lists + (lists + 1) / 2;
  unsigned* cand_i = reinterpret_cast<unsigned*>(cand_v + p.k * p.k);
  grid_launch_dependents();
  grid_dependency_wait();
  const int b = blockIdx.x;
  for (int w = warp; w < p.beams; w += kBeamThreads / 32) {
    const size_t at = (size_t(b) * p.beams + w) * p.chunks;
    float m = -INFINITY;
    for (int c = lane; c < p.chunks; c += 32) m = fmaxf(m, p.chunk_max[at + c]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    double s = 0.0;
    if (m != -INFINITY)
      for (int c = lane; c < p.chunks; c += 32)
        s += p.chunk_sum[at + c] * exp(double(p.chunk_max[at + c]) - double(m));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    // a row without a possible token, and a beam that is out, give -inf
    const float score = beam_logit(p.scores[size_t(b) * p.beams + w]);
    if (lane == 0) {
      s_off[w] = m == -INFINITY || score == -INFINITY ? -INFINITY : double(score) - log(s);
      s_top[w] = m == -INFINITY ? 0.f : m;
    }
  }
  if (tid == 0) {
    s_n = 0;
    s_tau_v = 0;
    s_tau_i = 0xffffffffu;
  }
  __syncthreads();
  const unsigned long long* keys = p.keys + size_t(b) * lists * p.k;
  // A candidate's score (logit - largest first: a row of lowest values, as
  // masks leave it, would swallow the rest)
  auto value = [&](int list, unsigned long long key) -> unsigned long long {
    const int w = list / p.chunks;
    return beam_order64(s_off[w] + (double(beam_value(unsigned(key >> 32))) - double(s_top[w])));
  };
  auto index = [&](int list, unsigned long long key) -> unsigned {
    return unsigned(list / p.chunks) * unsigned(p.vocab) + (0xffffffffu - unsigned(key));
  };
  auto before = [](unsigned long long va, unsigned ia, unsigned long long vb, unsigned ib) {
    return va > vb || (va == vb && ia < ib);
  };
  for (int l = tid; l < lists; l += kBeamThreads) {
    const unsigned long long key = keys[size_t(l) * p.k];
    head_v[l] = value(l, key);
    head_i[l] = index(l, key);
  }
  __syncthreads();
  for (int l = tid; l < lists; l += kBeamThreads) {  // the k-th best head
    const unsigned long long v = head_v[l];
    const unsigned id = head_i[l];
    int above = 0;
    for (int i = 0; i < lists; ++i) above += before(head_v[i], head_i[i], v, id);
    if (above == p.k - 1) {
      s_tau_v = v;
      s_tau_i = id;
    }
  }
  __syncthreads();
  const unsigned long long tau_v = s_tau_v;
  const unsigned tau_i = s_tau_i;
  for (int e = tid; e < lists * p.k; e += kBeamThreads) {
    const int l = e / p.k;
    if (before(tau_v, tau_i, head_v[l], head_i[l])) continue;  // a list behind the k best heads
    const unsigned long long key = keys[e];
    if (key == 0) continue;
    const unsigned long long v = value(l, key);
    const unsigned id = index(l, key);
    if (before(tau_v, tau_i, v, id)) continue;
    const int at = atomicAdd(&s_n, 1);
    cand_v[at] = v;
    cand_i[at] = id;
  }
  __syncthreads();
  const int n = s_n;
  for (int i = tid; i < n; i += kBeamThreads) {
    const unsigned long long v = cand_v[i];
    const unsigned id = cand_i[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += before(cand_v[j], cand_i[j], v, id);
    if (above < p.k) {
      const size_t at = size_t(b) * p.k + above;
      p.out_scores[at] = float(beam_value64(v));
      p.out_tokens[at] = int(id % unsigned(p.vocab));
      p.out_parents[at] = int(id / unsigned(p.vocab));
    }
  }
}

// ------------------------------------------------------------------- reorder

struct BeamReorderParams {
  int batch, beams_in, beams_out, max_pages, physical_pages, words;  // words: ceil(max_pages / 32)
  const int* parents;        // [batch, beams_out]: a beam of the same request, or -1
  const int* pages_in;       // [batch, beams_in, max_pages]
  const int* lengths_in;     // [batch, beams_in]
  const int* refcount_in;
  const int* free_stack_in;
  const int* free_count_in;
  int* refcount;             // (any of the state's outputs may be its input)
  int* free_stack;
  int* free_count;
  int* pages_out;            // [batch, beams_out, max_pages], not pages_in
  int* lengths_out;          // [batch, beams_out], not lengths_in
  unsigned* marks;           // workspace [batch * beams_in, words]
  int* children;             // workspace [batch * beams_in]
  unsigned* err;
};

constexpr int kReorderThreads = 256;
constexpr int kReleaseThreads = 1024;

// Blocks [0, row_blocks): a warp per (request, 32 columns) writes the new rows
// and marks, in each column, the last beam that holds a page whose reference
// count changes. The other blocks copy the state where it is not updated in
// place.
__global__ void __launch_bounds__(kReorderThreads)
    beam_rows_kernel(const BeamReorderParams p, int row_blocks) {
  __shared__ int s_child[kReorderThreads / 32][kBeamMax];
  __shared__ int s_parent[kReorderThreads / 32][kBeamMax];
  __shared__ int s_pages[kReorderThreads / 32][kBeamMax];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  if (int(blockIdx.x) >= row_blocks) {
    const int at = (int(blockIdx.x) - row_blocks) * kReorderThreads + tid;
    const int step = (int(gridDim.x) - row_blocks) * kReorderThreads;
    if (p.refcount != p.refcount_in)
      for (int i = at; i < p.physical_pages; i += step) p.refcount[i] = p.refcount_in[i];
    if (p.free_stack != p.free_stack_in)
      for (int i = at; i < p.physical_pages; i += step) p.free_stack[i] = p.free_stack_in[i];
    return;
  }
  const long long item = (long long)blockIdx.x * (kReorderThreads / 32) + warp;
  if (item >= (long long)p.batch * p.words) return;
  const int b = int(item / p.words), word = int(item % p.words), c = word * 32 + lane;
  int* child = s_child[warp];
  int* parent = s_parent[warp];
  int* held = s_pages[warp];  // page counts of the rows
  for (int r = lane; r < p.beams_in; r += 32) {
    int len = p.lengths_in[size_t(b) * p.beams_in + r];
    if (len < 0 || len > p.max_pages * kPageSize) {
      atomicOr(p.err, kErrLength);
      len = len < 0 ? 0 : p.max_pages * kPageSize;
    }
    held[r] = (len + kPageSize - 1) / kPageSize;
    child[r] = 0;
  }
  __syncwarp();
  for (int j = lane; j < p.beams_out; j += 32) {
    int r = p.parents[size_t(b) * p.beams_out + j];
    if (r < -1 || r >= p.beams_in) {
      atomicOr(p.err, kErrParent);
      r = -1;
    }
    parent[j] = r;
    if (r >= 0) atomicAdd(&child[r], 1);
    if (word == 0)
      p.lengths_out[size_t(b) * p.beams_out + j] = r < 0 ? 0 : p.lengths_in[size_t(b) * p.beams_in + r];
  }
  __syncwarp();
  if (word == 0)
    for (int r = lane; r < p.beams_in; r += 32) p.children[size_t(b) * p.beams_in + r] = child[r];
  const int* in = p.pages_in + size_t(b) * p.beams_in * p.max_pages + c;
  const bool col = c < p.max_pages;
  auto page_of = [&](int r) -> int {
    return col && c < held[r] ? in[size_t(r) * p.max_pages] : -1;
  };
  for (int j = 0; j < p.beams_out; ++j)
    if (col)
      p.pages_out[(size_t(b) * p.beams_out + j) * p.max_pages + c] = parent[j] < 0 ? -1 : page_of(parent[j]);
  for (int r = 0; r < p.beams_in; ++r) {
    const int page = page_of(r);
    bool mark = false;
    if (page >= 0 && page < p.physical_pages) {
      int net = child[r] - 1;
      mark = true;
      for (int o = 0; o < p.beams_in; ++o)
        if (o != r && page_of(o) == page) {
          net += child[o] - 1;
          if (o > r) mark = false;  // a later beam holds it too
        }
      mark = mark && net != 0;
    } else if (col && c < held[r]) {
      atomicOr(p.err, kErrPageRange);
    }
    const unsigned bits = __ballot_sync(0xffffffffu, mark);
    if (lane == 0) p.marks[(size_t(b) * p.beams_in + r) * p.words + word] = bits;
  }
}

// One block: applies the marked changes, then pushes the pages nobody holds
// any more in the order of their last release (row, then column). A page that
// beams of two requests held (a common prompt) may be marked in both: the
// later mark claims it, by writing its place into the zero reference count.
__global__ void __launch_bounds__(kReleaseThreads) beam_release_kernel(const BeamReorderParams p) {
  __shared__ int s_warp[kReleaseThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  const long long total = (long long)p.batch * p.beams_in * p.words;
  const long long per = (total + kReleaseThreads - 1) / kReleaseThreads;
  const long long w0 = min(total, tid * per), w1 = min(total, w0 + per);
  auto page_at = [&](long long w, int bit) -> int {
    return p.pages_in[size_t(w / p.words) * p.max_pages + size_t(w % p.words) * 32 + bit];
  };
  for (long long w = w0; w < w1; ++w) {
    for (unsigned bits = p.marks[w]; bits; bits &= bits - 1) {
      const int bit = __ffs(bits) - 1, page = page_at(w, bit);
      const long long row = w / p.words;
      const int b = int(row / p.beams_in), c = int(w % p.words) * 32 + bit;
      int net = 0;
      for (int r = 0; r < p.beams_in; ++r) {
        const size_t at = size_t(b) * p.beams_in + r;
        const int len = min(max(p.lengths_in[at], 0), p.max_pages * kPageSize);
        if (c < (len + kPageSize - 1) / kPageSize && p.pages_in[at * p.max_pages + c] == page)
          net += p.children[at] - 1;
      }
      atomicAdd(&p.refcount[page], net);
    }
  }
  __syncthreads();
  for (long long w = w0; w < w1; ++w) {  // keep the marks of pages that became free
    unsigned left = 0;
    const unsigned was = p.marks[w];
    for (unsigned bits = was; bits; bits &= bits - 1) {
      const int bit = __ffs(bits) - 1;
      if (*reinterpret_cast<volatile int*>(&p.refcount[page_at(w, bit)]) == 0) left |= 1u << bit;
    }
    if (left != was) p.marks[w] = left;
  }
  __syncthreads();
  for (long long w = w0; w < w1; ++w)
    for (unsigned bits = p.marks[w]; bits; bits &= bits - 1) {
      const int bit = __ffs(bits) - 1;
      atomicMin(&p.refcount[page_at(w, bit)], -int(w * 32 + bit) - 1);
    }
  __syncthreads();
  int mine = 0;
  for (long long w = w0; w < w1; ++w)
    for (unsigned bits = p.marks[w]; bits; bits &= bits - 1) {
      const int bit = __ffs(bits) - 1;
      mine += *reinterpret_cast<volatile int*>(&p.refcount[page_at(w, bit)]) == -int(w * 32 + bit) - 1;
    }
  int scan = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += up;
  }
  if (lane == 31) s_warp[warp] = scan;
  const int count = *p.free_count_in;
  __syncthreads();
  int before = scan - mine, freed = 0;
  for (int w = 0; w < kReleaseThreads / 32; ++w) {
    if (w < warp) before += s_warp[w];
    freed += s_warp[w];
  }
  for (long long w = w0; w < w1; ++w)
    for (unsigned bits = p.marks[w]; bits; bits &= bits - 1) {
      const int bit = __ffs(bits) - 1, page = page_at(w, bit);
      if (*reinterpret_cast<volatile int*>(&p.refcount[page]) != -int(w * 32 + bit) - 1) continue;
      const long long at = (long long)count + before++;
      if (at >= 0 && at < p.physical_pages)
        p.free_stack[at] = page;
      else
        atomicOr(p.err, kErrPageRange);
      p.refcount[page] = 0;
    }
  if (tid == 0) *p.free_count = min(count + freed, p.physical_pages);
}

}  // namespace bc
