// Beam search on the device: the k best (beam, token) pairs of every request
// (beam_segment_kernel, beam_merge_kernel) and the page tables and reference
// counts after the beams' new parents (beam_rows_kernel, beam_release_kernel).
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "bc_attn.cuh"

namespace bc {

constexpr int kBeamMax = 64;      // beams of a request
constexpr int kBeamMaxK = 64;     // pairs selected
constexpr int kBeamMaxVocab = 1 << 20;
constexpr int kBeamMergeThreads = 512;
constexpr int kBeamThreads = 256;
constexpr int kBeamLoads = 4;                         // 16-byte loads of a thread's step
constexpr int kBeamGroups = kBeamThreads / 2;         // two threads each

constexpr int kBeamSteps = 16;  // steps whose threads' maxima are kept

// Logits of one step of a block; the candidates there can be: those waiting (2 k +
// 32 at most before they are thinned) and those of one load by all threads.
__host__ __device__ constexpr int beam_tile(int type_bytes) {
  return kBeamThreads * kBeamLoads * (16 / type_bytes);
}
__host__ __device__ constexpr int beam_room(int k) { return 2 * k + 32 + kBeamThreads * 8; }
__host__ __device__ constexpr int beam_few(int k) {  // thinned (beam_thin)
  return k * ((beam_room(k) + kBeamThreads - 1) / kBeamThreads);
}
__host__ __device__ constexpr size_t beam_smem(int k) {
  return size_t(beam_room(k) + beam_few(k)) * 8 + size_t(kBeamSteps) * kBeamThreads * 4;
}

enum BeamType : int { kBeamF16 = 0, kBeamBF16 = 1, kBeamF32 = 2 };

// A score as the search sees it: NaN counts as -inf, +inf as the largest number.
__device__ __forceinline__ float beam_score(float x) {
  return fminf(fmaxf(x, -INFINITY), 3.402823466e38f);
}

// Logits likewise (NaN is never chosen before a number, +inf is their type's
// largest), two 16-bit ones at a time; and the larger of two words' logits.
__device__ __forceinline__ uint32_t beam_clean(uint32_t x, const float*) {
  return __float_as_uint(beam_score(__uint_as_float(x)));
}
__device__ __forceinline__ uint32_t beam_clean(uint32_t x, const __half*) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tmax.f16x2 t, %1, %2;\n\tmin.f16x2 %0, t, %3;\n\t}"
      : "=r"(r) : "r"(x), "r"(0xfc00fc00u), "r"(0x7bff7bffu));
  return r;
}
__device__ __forceinline__ uint32_t beam_clean(uint32_t x, const __nv_bfloat16*) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tmax.bf16x2 t, %1, %2;\n\tmin.bf16x2 %0, t, %3;\n\t}"
      : "=r"(r) : "r"(x), "r"(0xff80ff80u), "r"(0x7f7f7f7fu));
  return r;
}
__device__ __forceinline__ uint32_t beam_max(uint32_t x, uint32_t y, const float*) {
  return __float_as_uint(fmaxf(__uint_as_float(x), __uint_as_float(y)));
}
__device__ __forceinline__ uint32_t beam_max(uint32_t x, uint32_t y, const __half*) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
__device__ __forceinline__ uint32_t beam_max(uint32_t x, uint32_t y, const __nv_bfloat16*) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
// Logit i of a word.
__device__ __forceinline__ float beam_float(uint32_t w, int, const float*) { return __uint_as_float(w); }
__device__ __forceinline__ float beam_float(uint32_t w, int i, const __half*) {
  const float2 f = unpack_half2(w);
  return i ? f.y : f.x;
}
__device__ __forceinline__ float beam_float(uint32_t w, int i, const __nv_bfloat16*) {
  return __uint_as_float(i ? w & 0xffff0000u : w << 16);
}

__device__ __forceinline__ float beam_one(float x) { return beam_score(x); }
__device__ __forceinline__ float beam_one(__half x) {
  return beam_float(beam_clean(uint32_t(__half_as_ushort(x)), static_cast<const __half*>(nullptr)), 0,
                    static_cast<const __half*>(nullptr));
}
__device__ __forceinline__ float beam_one(__nv_bfloat16 x) {
  return beam_float(
      beam_clean(uint32_t(__bfloat16_as_ushort(x)), static_cast<const __nv_bfloat16*>(nullptr)), 0,
      static_cast<const __nv_bfloat16*>(nullptr));
}

// Keys: larger value first, then the lower index. Unique, so selection never
// meets a tie. (-0 is +0: equal logits are equal in their key's value.)
__device__ __forceinline__ unsigned beam_order(float x) {
  const unsigned u = __float_as_uint(x + 0.f);
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

// The 16 bytes from byte `by` (below 16) of 32 on.
__device__ __forceinline__ uint4 beam_shift(uint4 lo, uint4 hi, unsigned by) {
  const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  uint32_t a[6], b[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) a[i] = by & 8u ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) b[i] = by & 4u ? a[i + 1] : a[i];
  const unsigned bits = (by & 3u) * 8u;
  return make_uint4(__funnelshift_r(b[0], b[1], bits), __funnelshift_r(b[1], b[2], bits),
                    __funnelshift_r(b[2], b[3], bits), __funnelshift_r(b[3], b[4], bits));
}

struct BeamSelectParams {
  int batch, beams, vocab, k;
  int segments, segment;  // blocks of a row, their steps' logits (a multiple of the step)
  const void* logits;
  long long row_stride;  // elements between two beams' rows
  const float* scores;   // [batch, beams]
  float* out_scores;     // [batch, k]
  int* out_tokens;
  int* out_parents;
  // workspace, per (row, segment): the k best keys in order (0 past the
  // segment's logits), the largest logit and the sum of exp(x - largest)
  unsigned long long* keys;  // [rows, segments, k]
  float* seg_max;            // [rows, segments]
  double* seg_sum;           // [rows, segments]
};

// What the thinning of candidates needs beside them.
struct BeamThin {
  unsigned long long best[kBeamThreads];
  unsigned long long out[kBeamMaxK];
  unsigned long long tau;
  int count;
};

// Keeps the k best of the n candidates in `cand` (in order, at its front), for
// all threads of the block; returns how many there are. Many candidates are
// thinned into `few` first: at most k threads hold keys at or above the k-th
// largest of the threads' maxima.
__device__ __noinline__ int beam_thin(unsigned long long* cand, unsigned long long* few, BeamThin& t,
                                      int n, int k) {
  const int tid = threadIdx.x;
  const unsigned long long* from = cand;
  if (n > 2 * kBeamThreads) {
    unsigned long long mx = 0;
    for (int i = tid; i < n; i += kBeamThreads) mx = cand[i] > mx ? cand[i] : mx;
    t.best[tid] = mx;
    if (tid == 0) t.count = 0;
    __syncthreads();
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kBeamThreads; ++i) above += t.best[i] > mx;
    if (above == k - 1) t.tau = mx;  // (keys are unique: one thread)
    __syncthreads();
    if (mx >= t.tau)
      for (int i = tid; i < n; i += kBeamThreads)
        if (cand[i] >= t.tau) few[atomicAdd(&t.count, 1)] = cand[i];
    __syncthreads();
    n = t.count;
    from = few;
  }
  for (int i = tid; i < n; i += kBeamThreads) {  // rank by counting
    const unsigned long long mine = from[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) above += from[j] > mine;
    if (above < k) t.out[above] = mine;
  }
  __syncthreads();
  n = min(n, k);
  if (tid < n) cand[tid] = t.out[tid];
  __syncthreads();
  return n;
}

// One block per segment of a row. One pass of 16-byte loads, the next step's in flight
// (32 x 8 x 131071 BF16 logits, rows off the 16-byte boundaries: 37 us, 22 % of HBM; a
// segment's fixed work and those rows' loads bound it), in which every thread keeps its
// largest logit (the first such) and its sum of exp(x - largest) under its running
// maximum, no barrier between the steps. The k-th largest of 128 thread pairs' best keys bounds the segment's k best,
// which lie in k pairs: those few threads look again (from L2) at the steps whose
// maxima, kept in shared memory, reach the bound and list what passes. Should the
// list run over, they go through all steps a load at a time, thinning it on the way.
// The sum takes ex2.approx of (x - largest) log2(e): relative error 2^-22 and the
// argument's, none for the thread's largest logit itself; a step's 16 or 32 terms are
// added in FP32, the steps and threads in 64 bits, since the order of two beams'
// candidates hangs on the last digits.
template <typename T>
__global__ void __launch_bounds__(kBeamThreads, 4) beam_segment_kernel(const BeamSelectParams p) {
  constexpr float kLog2E = 1.4426950408889634f;
  // a thread's logits of a step: 16 words, PW to a word, VEC to a load
  constexpr int PW = 4 / int(sizeof(T)), VEC = 4 * PW, PT = VEC * kBeamLoads, TILE = beam_tile(sizeof(T));
  constexpr const T* kType = nullptr;
  extern __shared__ unsigned long long beam_cand[];  // [beam_room], [beam_few], step maxima
  __shared__ BeamThin s_thin;
  __shared__ float s_max[kBeamThreads / 32];
  __shared__ double s_sum[kBeamThreads / 32];
  __shared__ int s_n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_launch_dependents();
  if (tid == 0) {
    s_n = 0;
    s_thin.tau = 0;
  }
  grid_dependency_wait();
  const int row = blockIdx.x / p.segments, seg = blockIdx.x % p.segments;
  const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
  // Threads take tokens by their numbers wherever the row lies, so that rows alike are
  // summed alike, to the last bit: pairs of such beams are equal, and ordered by their
  // index. A row off the 16-byte boundaries puts its vectors together from the two
  // aligned ones that hold them (each of which holds a logit of the row).
  const unsigned mis = unsigned(reinterpret_cast<uintptr_t>(x) & 15);  // bytes
  const uint4* lines = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x) - mis);
  const int w0 = seg * p.segment, w1 = min(w0 + p.segment, p.vocab);
  const float score = p.scores[row];
  auto load = [&](int w, uint32_t (&raw)[16]) {
#pragma unroll
    for (int j = 0; j < kBeamLoads; ++j) {
      const int at = w + (j * kBeamThreads + tid) * VEC;
      uint4 v;
      if (at + VEC <= p.vocab) {
        v = __ldcs(lines + at / VEC);
        if (mis) v = beam_shift(v, __ldcs(lines + at / VEC + 1), mis);
      } else {  // a vector across the row's end: its own logits alone
        T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = at + i < p.vocab ? x[at + i] : T(-INFINITY);
        v = *reinterpret_cast<const uint4*>(e);
      }
      raw[4 * j] = v.x;
      raw[4 * j + 1] = v.y;
      raw[4 * j + 2] = v.z;
      raw[4 * j + 3] = v.w;
    }
  };
  // The same for the stream, where the words' place is settled once a step.
  auto words = [&](auto skip, int w, uint32_t (&raw)[16]) {
    constexpr int S = decltype(skip)::value;  // whole words of `mis`
    const unsigned bits = (mis & 3u) * 8u;
#pragma unroll
    for (int j = 0; j < kBeamLoads; ++j) {
      const int at = w + (j * kBeamThreads + tid) * VEC;
      const uint4 lo = __ldcs(lines + at / VEC), hi = __ldcs(lines + at / VEC + 1);
      const uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        raw[4 * j + i] = sizeof(T) == 4 ? v[i + S] : __funnelshift_r(v[i + S], v[i + S + 1], bits);
    }
  };
  auto fetch = [&](int w, uint32_t (&raw)[16]) {
    if (mis == 0 || w + TILE > p.vocab) {
      load(w, raw);
    } else {
      switch (mis >> 2) {
        case 0: words(std::integral_constant<int, 0>{}, w, raw); break;
        case 1: words(std::integral_constant<int, 1>{}, w, raw); break;
        case 2: words(std::integral_constant<int, 2>{}, w, raw); break;
        default: words(std::integral_constant<int, 3>{}, w, raw);
      }
    }
  };
  uint32_t raw[16], next[16];
  if (w0 < w1) fetch(w0, raw);
  // A beam that is out: all its pairs score -inf, so its first tokens are its best,
  // whatever their logits. (Looked at with the first logits on their way: beside
  // them, the score costs no wait of its own.)
  if (beam_score(score) == -INFINITY) {
    for (int i = tid; i < p.k; i += kBeamThreads)
      p.keys[size_t(blockIdx.x) * p.k + i] =
          w0 + i < w1 ? beam_key(-INFINITY, unsigned(w0 + i)) : 0ull;
    if (tid == 0) {
      p.seg_max[blockIdx.x] = -INFINITY;
      p.seg_sum[blockIdx.x] = 0.0;
    }
    return;
  }
  auto val = [&](int j) { return beam_float(raw[j / PW], j % PW, kType); };
  // the thread's logits at or above `bound`, a bit each
  auto at_or_above = [&](float bound) -> uint32_t {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < PT; ++j) bits |= val(j) >= bound ? 1u << j : 0u;
    return bits;
  };
  auto clean = [&]() -> float {  // raw made ready; its largest logit
#pragma unroll
    for (int i = 0; i < 16; ++i) raw[i] = beam_clean(raw[i], kType);
    uint32_t big = raw[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) big = beam_max(big, raw[i], kType);
    return fmaxf(beam_float(big, 0, kType), beam_float(big, PW - 1, kType));
  };
  auto place = [&](int w, int j) { return w + (j / VEC * kBeamThreads + tid) * VEC + j % VEC; };
  const int room = beam_room(p.k);
  unsigned long long* few = beam_cand + room;
  float* step_max = reinterpret_cast<float*>(few + beam_few(p.k)) + tid;  // [step * kBeamThreads]
  float m = -INFINITY;
  double sum = 0.0;
  int top = w0;  // the first step with the largest logit
  for (int w = w0, i = 0; w < w1; w += TILE, ++i) {
    if (w + TILE < w1) fetch(w + TILE, next);
    const float mx = clean();
    if (i < kBeamSteps) step_max[i * kBeamThreads] = mx;
    if (mx > m) {
      sum *= m == -INFINITY ? 0.0 : double(expf(m - mx));
      m = mx;
      top = w;
    }
    const float base = m == -INFINITY ? 0.f : m;
    uint64_t e = 0;  // (two zeros)
#pragma unroll
    for (int j = 0; j < PT; j += 2) {
      const float2 d = pair_floats(mul2(add2(pair_of(val(j), val(j + 1)), pair_of(-base, -base)),
                                        pair_of(kLog2E, kLog2E)));
      e = add2(e, pair_of(fast_exp2(d.x), fast_exp2(d.y)));
    }
    sum += double(pair_floats(e).x + pair_floats(e).y);
#pragma unroll
    for (int i = 0; i < 16; ++i) raw[i] = next[i];
  }
  // the thread's best key (0: it has no logit of the row)
  unsigned long long best = 0;
  for (int w = top; w < w1 && best == 0; w += TILE) {
    load(w, raw);
    clean();
    for (uint32_t bits = at_or_above(m); bits; bits &= bits - 1) {
      const int at = place(w, __ffs(bits) - 1);
      if (at < w1) {
        best = beam_key(m, unsigned(at));
        break;
      }
    }
    if (m != -INFINITY) break;  // (only fillers at the row's ends can be passed over)
  }
  // the bound: both threads of a pair count against half the pairs
  unsigned long long pair = __shfl_xor_sync(0xffffffffu, best, 1);
  pair = pair > best ? pair : best;
  s_thin.best[tid] = pair;
  __syncthreads();
  {
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kBeamGroups / 2; ++i)
      above += s_thin.best[((tid & 1) * (kBeamGroups / 2) + i) * 2] > pair;
    above += __shfl_xor_sync(0xffffffffu, above, 1);
    if (above == p.k - 1 && pair != 0 && (tid & 1) == 0) s_thin.tau = pair;
  }
  __syncthreads();
  unsigned long long tau = s_thin.tau;
  // lists the thread's logits of the step at w, of the loads in `of`, whose keys reach
  // tau; true when there are more than `most` in the list
  auto list_step = [&](int w, uint32_t of, int most) -> bool {
    bool over = false;
    load(w, raw);
    const float bound = tau == 0 ? -INFINITY : beam_value(unsigned(tau >> 32));
    if (clean() >= bound)
      for (uint32_t bits = at_or_above(bound) & of; bits; bits &= bits - 1) {
        const int at = place(w, __ffs(bits) - 1);
        if (at >= w1) continue;
        // (few: read again, rather than picked out of the registers)
        const unsigned long long key = beam_key(beam_one(x[at]), unsigned(at));
        if (key < tau) continue;
        const int i = atomicAdd(&s_n, 1);
        if (i < room) beam_cand[i] = key;
        over = over || i >= most;
      }
    return over;
  };
  const bool look = best >= tau && best != 0;
  if (look) {
    const float bound = tau == 0 ? -INFINITY : beam_value(unsigned(tau >> 32));
    for (int w = w0, i = 0; w < w1; w += TILE, ++i)
      if (i >= kBeamSteps || step_max[i * kBeamThreads] >= bound) list_step(w, 0xffffffffu, room);
  }
  __syncthreads();
  int n = s_n;
  __syncthreads();
  if (n > room) {
    if (tid == 0) s_n = 0;
    __syncthreads();
    for (int w = w0; w < w1; w += TILE)
      for (int j = 0; j < kBeamLoads; ++j) {
        const uint32_t of = (VEC == 8 ? 0xffu : 0xfu) << (j * VEC);
        const bool over = look && list_step(w, of, 2 * p.k + 32);
        // (the answer has to be the block's: s_n may have moved on for some)
        if (__syncthreads_or(over)) {
          n = beam_thin(beam_cand, few, s_thin, s_n, p.k);
          if (n == p.k) tau = beam_cand[n - 1] + 1;  // only better ones from now on
          if (tid == 0) s_n = n;
          __syncthreads();
        }
      }
    n = s_n;
    __syncthreads();
  }
  n = beam_thin(beam_cand, few, s_thin, n, p.k);
  const size_t at = size_t(blockIdx.x) * p.k;
  for (int i = tid; i < p.k; i += kBeamThreads) p.keys[at + i] = i < n ? beam_cand[i] : 0ull;
  // the segment's maximum and sum
  float bm = m;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, d));
  if (lane == 0) s_max[warp] = bm;
  __syncthreads();
  bm = s_max[0];
#pragma unroll
  for (int w = 1; w < kBeamThreads / 32; ++w) bm = fmaxf(bm, s_max[w]);
  sum = m == -INFINITY ? 0.0 : sum * exp(double(m) - double(bm));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    double total = 0.0;
    for (int w = 0; w < kBeamThreads / 32; ++w) total += s_sum[w];
    p.seg_max[blockIdx.x] = bm;
    p.seg_sum[blockIdx.x] = total;
  }
}

// One block per request: the rows' log sums, then the k best of all segments'
// lists. Lists are sorted, so the k best lie in the k lists with the best
// heads: at most k*k candidates.
__global__ void __launch_bounds__(kBeamMergeThreads) beam_merge_kernel(const BeamSelectParams p) {
  extern __shared__ unsigned long long beam_lists[];
  __shared__ double s_off[kBeamMax];
  __shared__ float s_top[kBeamMax];
  __shared__ int s_n;
  __shared__ unsigned long long s_tau_v;
  __shared__ unsigned s_tau_i;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lists = p.beams * p.segments;
  unsigned long long* head_v = beam_lists;                  // [lists] order of the head's score
  unsigned* head_i = reinterpret_cast<unsigned*>(head_v + lists);  // [lists] its beam*vocab + token
  unsigned long long* cand_v = head_v + lists + (lists + 1) / 2;
  unsigned* cand_i = reinterpret_cast<unsigned*>(cand_v + p.k * p.k);
  grid_launch_dependents();
  grid_dependency_wait();
  const int b = blockIdx.x;
  for (int w = warp; w < p.beams; w += kBeamMergeThreads / 32) {
    const size_t at = (size_t(b) * p.beams + w) * p.segments;
    float m = -INFINITY;
    for (int c = lane; c < p.segments; c += 32) m = fmaxf(m, p.seg_max[at + c]);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    double s = 0.0;
    if (m != -INFINITY)
      for (int c = lane; c < p.segments; c += 32)
        s += p.seg_sum[at + c] * exp(double(p.seg_max[at + c]) - double(m));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    // a row without a possible token, and a beam that is out, give -inf
    const float score = beam_score(p.scores[size_t(b) * p.beams + w]);
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
    const int w = list / p.segments;
    return beam_order64(s_off[w] + (double(beam_value(unsigned(key >> 32))) - double(s_top[w])));
  };
  auto index = [&](int list, unsigned long long key) -> unsigned {
    return unsigned(list / p.segments) * unsigned(p.vocab) + (0xffffffffu - unsigned(key));
  };
  auto before = [](unsigned long long va, unsigned ia, unsigned long long vb, unsigned ib) {
    return va > vb || (va == vb && ia < ib);
  };
  for (int l = tid; l < lists; l += kBeamMergeThreads) {
    const unsigned long long key = keys[size_t(l) * p.k];
    head_v[l] = value(l, key);  // (every segment has a logit: no list is empty)
    head_i[l] = index(l, key);
  }
  __syncthreads();
  for (int l = tid; l < lists; l += kBeamMergeThreads) {  // the k-th best head
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
  for (int e = tid; e < lists * p.k; e += kBeamMergeThreads) {
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
  for (int i = tid; i < n; i += kBeamMergeThreads) {
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
  unsigned* err;
};

constexpr int kReorderWarps = 4;
constexpr int kReleaseThreads = 1024;
constexpr int kReleaseList = 256;  // freed pages of a warp that fit in shared memory
constexpr size_t kReleaseSmem = size_t(kReleaseThreads / 32) * kReleaseList * sizeof(int2);

// The state's copies, where it is not updated in place.
__global__ void __launch_bounds__(256) pool_copy_kernel(int n, const int* __restrict__ a, int* a_out,
                                                        const int* __restrict__ b, int* b_out) {
  grid_launch_dependents();
  grid_dependency_wait();
  for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
    if (a_out != a) a_out[i] = a[i];
    if (b_out != b) b_out[i] = b[i];
  }
}

// A warp per (request, 32 columns): the old entries are read once, the new rows
// written; a page's reference count changes by its holders' children less one
// each, once per column, and where that is a loss the last beam holding it is
// marked (the page may be free now). Most columns are one page held by all beams,
// as many before as after: nothing to do.
__global__ void __launch_bounds__(kReorderWarps * 32) beam_rows_kernel(const BeamReorderParams p) {
  __shared__ int s_child[kReorderWarps][kBeamMax];
  __shared__ int s_parent[kReorderWarps][kBeamMax];
  __shared__ int s_pages[kReorderWarps][kBeamMax][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  const unsigned item = blockIdx.x * kReorderWarps + warp;  // (words of all marks: below 2^26)
  if (item >= unsigned(p.batch) * p.words) return;
  const int b = int(item / unsigned(p.words)), word = int(item % unsigned(p.words)), c = word * 32 + lane;
  int* child = s_child[warp];
  int* parent = s_parent[warp];
  int (*page)[32] = s_pages[warp];
  const bool col = c < p.max_pages;
  const int* in = p.pages_in + size_t(b) * p.beams_in * p.max_pages + c;
  bool bad_page = false;
#pragma unroll 8
  for (int r = 0; r < p.beams_in; ++r) {
    const int raw = p.lengths_in[size_t(b) * p.beams_in + r];
    const int len = min(max(raw, 0), p.max_pages * kPageSize);
    if (raw != len && lane == 0) atomicOr(p.err, kErrLength);
    int id = -1;
    if (col && c < (len + kPageSize - 1) / kPageSize) {
      id = in[size_t(r) * p.max_pages];
      bad_page |= id < 0 || id >= p.physical_pages;
    }
    page[r][lane] = id;
  }
  if (bad_page) atomicOr(p.err, kErrPageRange);
  for (int r = lane; r < p.beams_in; r += 32) child[r] = 0;
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
  if (col)
    for (int j = 0; j < p.beams_out; ++j)
      p.pages_out[(size_t(b) * p.beams_out + j) * p.max_pages + c] =
          parent[j] < 0 ? -1 : page[parent[j]][lane];
  // (children of all rows less rows: the change of a page that all hold)
  int all = -p.beams_in;
  for (int r = 0; r < p.beams_in; ++r) all += child[r];
  bool same = true;
  for (int r = 1; r < p.beams_in; ++r) same = same && page[r][lane] == page[0][lane];
  const bool quiet = same && (all == 0 || page[0][lane] < 0);
  const bool none = __all_sync(0xffffffffu, quiet);
  for (int r = 0; r < p.beams_in; ++r) {
    bool mark = false;
    const int id = page[r][lane];
    if (!quiet && id >= 0 && id < p.physical_pages) {
      int net = child[r] - 1;
      bool last = true;
      for (int o = 0; o < p.beams_in; ++o)
        if (o != r && page[o][lane] == id) {
          net += child[o] - 1;
          last = last && o < r;
        }
      if (last && net != 0) atomicAdd(&p.refcount[id], net);
      mark = last && net < 0;
    }
    const unsigned bits = none ? 0u : __ballot_sync(0xffffffffu, mark);
    if (lane == 0) p.marks[(size_t(b) * p.beams_in + r) * p.words + word] = bits;
  }
}

// One block: of the marked pages, those that nobody holds any more are pushed in
// the order of their last release (row, then column). A page that beams of two
// requests held (a common prompt) may be marked in both: the later mark claims it,
// by writing its place into the zero reference count. Every warp takes a run of
// words of the marks, its freed pages listed in order in shared memory; where a
// list runs over, all warps go through the marks themselves instead.
__global__ void __launch_bounds__(kReleaseThreads) beam_release_kernel(const BeamReorderParams p) {
  extern __shared__ int2 release_list[];
  __shared__ int s_warp[kReleaseThreads / 32];
  __shared__ int s_over;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kWarps = kReleaseThreads / 32;
  grid_launch_dependents();
  if (tid == 0) s_over = 0;
  grid_dependency_wait();
  __syncthreads();
  const int total = p.batch * p.beams_in * p.words;  // (below 2^26)
  const int per = (total + kWarps - 1) / kWarps;
  const int w0 = min(total, warp * per), w1 = min(total, w0 + per);
  auto page_at = [&](int w, int bit) -> int {
    const unsigned row = unsigned(w) / unsigned(p.words);
    return p.pages_in[size_t(row) * p.max_pages + (unsigned(w) - row * p.words) * 32 + bit];
  };
  auto count_of = [&](int page) { return *reinterpret_cast<volatile int*>(&p.refcount[page]); };
  const int count = *p.free_count_in;

  // the marked pages that became free: their marks stay, and they are listed
  int2* list = release_list + warp * kReleaseList;  // (place, page)
  int n = 0;
  unsigned ahead = w0 + lane < w1 ? p.marks[w0 + lane] : 0u;
  for (int g = w0; g < w1; g += 32) {
    const unsigned word = ahead;
    ahead = g + 32 + lane < w1 ? p.marks[g + 32 + lane] : 0u;
    unsigned some = __ballot_sync(0xffffffffu, word != 0u);
    while (some) {  // eight words of marks at a time, a lane a bit
      int src[8], page[8], rc[8];
      unsigned bits[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        src[i] = some ? __ffs(some) - 1 : -1;
        bits[i] = __shfl_sync(0xffffffffu, word, max(src[i], 0));
        if (src[i] < 0) bits[i] = 0u;
        some &= some - 1;
        page[i] = (bits[i] >> lane) & 1u ? page_at(g + src[i], lane) : -1;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) rc[i] = page[i] >= 0 ? count_of(page[i]) : 1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned left = __ballot_sync(0xffffffffu, rc[i] == 0);
        const int at = n + __popc(left & ((1u << lane) - 1));
        if (rc[i] == 0 && at < kReleaseList) list[at] = make_int2((g + src[i]) * 32 + lane, page[i]);
        n += __popc(left);
        if (lane == 0 && src[i] >= 0 && left != bits[i]) p.marks[g + src[i]] = left;
      }
    }
  }
  if (n > kReleaseList && lane == 0) s_over = 1;
  __syncthreads();
  const bool listed = s_over == 0;
  auto push = [&](long long at, int page) {
    if (at >= 0 && at < p.physical_pages)
      p.free_stack[at] = page;
    else
      atomicOr(p.err, kErrPageRange);
    p.refcount[page] = 0;
  };
  int freed = 0;
  // the pushes of the warps before this one
  auto before_of = [&](int mine) -> int {
    if (lane == 0) s_warp[warp] = mine;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_warp[w];
      freed += s_warp[w];
    }
    return before;
  };
  if (listed) {  // (a lane's entries in registers: the phases' accesses overlap)
    constexpr int kMine = kReleaseList / 32;
    int2 e[kMine];
    unsigned wins[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const bool in = i * 32 + lane < n;
      e[i] = in ? list[i * 32 + lane] : make_int2(-1, -1);
      if (in) atomicMin(&p.refcount[e[i].y], -e[i].x - 1);
    }
    __syncthreads();
    int now[kMine], mine = 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) now[i] = e[i].x >= 0 ? count_of(e[i].y) : 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      wins[i] = __ballot_sync(0xffffffffu, e[i].x >= 0 && now[i] == -e[i].x - 1);
      mine += __popc(wins[i]);
    }
    long long at = (long long)count + before_of(mine);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      if ((wins[i] >> lane) & 1u) push(at + __popc(wins[i] & ((1u << lane) - 1)), e[i].y);
      at += __popc(wins[i]);
    }
  } else {
    // (this lane's bit of each of the warp's words, in order)
    auto each = [&](auto&& f) {
      for (int w = w0; w < w1; ++w) {
        const unsigned bits = p.marks[w];
        if (bits == 0u) continue;
        const bool in = (bits >> lane) & 1u;
        f(in, w * 32 + lane, in ? page_at(w, lane) : 0);
      }
    };
    each([&](bool in, int place, int page) {
      if (in) atomicMin(&p.refcount[page], -place - 1);
    });
    __syncthreads();
    int mine = 0;
    each([&](bool in, int place, int page) {
      mine += __popc(__ballot_sync(0xffffffffu, in && count_of(page) == -place - 1));
    });
    long long at = (long long)count + before_of(mine);
    each([&](bool in, int place, int page) {
      const bool won = in && count_of(page) == -place - 1;
      const unsigned wins = __ballot_sync(0xffffffffu, won);
      if (won) push(at + __popc(wins & ((1u << lane) - 1)), page);
      at += __popc(wins);
    });
  }
  if (tid == 0) *p.free_count = int(min((long long)count + freed, (long long)p.physical_pages));
}

}  // namespace bc
