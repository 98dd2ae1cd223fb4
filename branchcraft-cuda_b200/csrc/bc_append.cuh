// New tokens into the paged cache: the page bookkeeping that gives every new
// token a slot (append_plan_kernel, append_expand_kernel) and the copy of its
// K/V row there (append_kv_kernel).
//
// The bookkeeping follows the page pool's rules (bc_cow.PagePool), sequence b
// taking new_tokens[b] tokens after its lengths[b] in batch order:
//   * a partial last page that others hold too (refcount > 1) is cloned into a
//     popped page, which replaces it in the row, and loses a reference;
//   * pages are popped until the row covers the new length, with refcount 1.
// A clone never frees a page, so nothing is pushed and the sequential replay
// has a closed form: among the h sequences of the batch that write into the
// same shared page, all clone it while somebody else holds it (h < refcount);
// when they are all its holders (h == refcount) the last of them in batch
// order finds itself alone and writes in place. The pops are the free stack's
// entries below its top at offsets given by a prefix sum.
#pragma once

#include "bc_attn.cuh"

namespace bc {

constexpr int kAppendMaxBatch = 4096;
constexpr int kPlanThreads = 1024;
constexpr int kExpandThreads = 256;
constexpr int kExpandTokens = 1024;  // tokens of one block of the expansion

enum AppendStatus : int {
  kAppendOk = 0,
  kAppendBadCount = 1,   // a count below zero, or more tokens than max_tokens
  kAppendExhausted = 2,  // not enough free pages
  kAppendBadTable = 3,   // lengths, page ids, refcounts or the stack are malformed
};

struct AppendPlanParams {
  int batch, physical_pages, max_pages_in, max_pages_out, max_tokens;
  const int* pages_in;       // [batch, max_pages_in]
  const int* lengths_in;     // [batch]
  const int* new_tokens;     // [batch]
  const int* refcount_in;    // [P]
  const int* free_stack_in;  // [P]
  const int* free_count_in;  // [1]
  int* refcount;             // (any of the state's outputs may be its input)
  int* free_stack;
  int* free_count;
  int* pages_out;            // [batch, max_pages_out] (may be pages_in at equal width)
  int* lengths_out;
  int* query_start;          // [batch + 1]
  int* slot_map;             // [max_tokens]
  int* positions;            // [max_tokens]
  int* clones;               // [3, batch]: source page, destination page, slots to copy
  int* counts;               // [3]: tokens, clones, status
  int* scratch;              // [batch + 1]: first pop * 2 + clone flag (-1: no plan), then the
                             // old free count
};

// Shared memory of the planner: the hash table of shared last pages (page,
// members, last member, smallest and largest length) with two entries a
// sequence, then one word a sequence.
__host__ __device__ inline int append_hash_size(int batch) {
  int n = 64;
  while (n < 2 * batch) n *= 2;
  return n;
}
__host__ __device__ inline size_t append_plan_smem_bytes(int batch) {
  return (size_t(append_hash_size(batch)) * 5 + size_t(batch)) * sizeof(int);
}

struct AppendSums {
  long long tokens, pops;
  int clones;
};

__device__ __forceinline__ AppendSums append_add(AppendSums a, const AppendSums& b) {
  a.tokens += b.tokens;
  a.pops += b.pops;
  a.clones += b.clones;
  return a;
}

__device__ __forceinline__ AppendSums append_shfl_up(const AppendSums& a, int d) {
  AppendSums r;
  r.tokens = __shfl_up_sync(0xffffffffu, a.tokens, d);
  r.pops = __shfl_up_sync(0xffffffffu, a.pops, d);
  r.clones = __shfl_up_sync(0xffffffffu, a.clones, d);
  return r;
}

// Block 0 plans; the other blocks copy the state where it is not updated in
// place, so that the expansion, which follows, only has to change it.
__global__ void __launch_bounds__(kPlanThreads) append_plan_kernel(const AppendPlanParams p) {
  extern __shared__ int plan_smem[];
  const int tid = threadIdx.x;
  grid_launch_dependents();
  grid_dependency_wait();
  if (blockIdx.x > 0) {
    const int at = (int(blockIdx.x) - 1) * kPlanThreads + tid, step = (int(gridDim.x) - 1) * kPlanThreads;
    if (p.refcount != p.refcount_in)
      for (int i = at; i < p.physical_pages; i += step) p.refcount[i] = p.refcount_in[i];
    if (p.free_stack != p.free_stack_in)
      for (int i = at; i < p.physical_pages; i += step) p.free_stack[i] = p.free_stack_in[i];
    return;
  }
  const int hsize = append_hash_size(p.batch), hmask = hsize - 1;
  int* h_page = plan_smem;
  int* h_members = h_page + hsize;
  int* h_last = h_members + hsize;
  int* h_min = h_last + hsize;
  int* h_max = h_min + hsize;
  int* entry = h_max + hsize;  // [batch] hash entry of a sequence with a shared last page, or -1
  __shared__ int s_bad_count, s_bad_table, s_status, s_free;
  __shared__ AppendSums s_warp[kPlanThreads / 32];
  if (tid == 0) {
    s_bad_count = s_bad_table = 0;
    s_free = *p.free_count_in;
  }
  for (int i = tid; i < hsize; i += kPlanThreads) {
    h_page[i] = -1;
    h_members[i] = 0;
    h_last[i] = -1;
    h_min[i] = 0x7fffffff;
    h_max[i] = -1;
  }
  __syncthreads();

  // Every sequence's row, checked; those whose partial last page is shared
  // meet in the hash table.
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    const int len = p.lengths_in[b], n = p.new_tokens[b];
    int e = -1;
    if (n < 0 || n > p.max_tokens) {
      s_bad_count = 1;
    } else if (len < 0 || len > p.max_pages_in * kPageSize ||
               ((long long)len + n + kPageSize - 1) / kPageSize > p.max_pages_out) {
      s_bad_table = 1;
    } else if (n > 0 && len % kPageSize != 0) {
      const int page = p.pages_in[size_t(b) * p.max_pages_in + len / kPageSize];
      const int rc = page >= 0 && page < p.physical_pages ? p.refcount_in[page] : 0;
      if (rc < 1) {
        s_bad_table = 1;
      } else if (rc > 1) {
        e = int((unsigned(page) * 2654435761u) >> 7) & hmask;
        for (;;) {  // (half the table stays empty: a free entry is found)
          const int had = atomicCAS(&h_page[e], -1, page);
          if (had == -1 || had == page) break;
          e = (e + 1) & hmask;
        }
        atomicAdd(&h_members[e], 1);
        atomicMax(&h_last[e], b);
        atomicMin(&h_min[e], len);
        atomicMax(&h_max[e], len);
      }
    }
    entry[b] = e;
  }
  __syncthreads();
  const bool bad = s_bad_count != 0 || s_bad_table != 0;

  // A thread's run of consecutive sequences, then sums over the block.
  const int per = (p.batch + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  auto clones_page = [&](int b, int page_rc) -> bool {
    const int e = entry[b];
    return h_members[e] < page_rc || h_last[e] != b;
  };
  auto one = [&](int b) -> AppendSums {
    const int len = p.lengths_in[b], n = p.new_tokens[b];
    int clone = 0;
    if (entry[b] >= 0) {
      const int e = entry[b], rc = p.refcount_in[h_page[e]];
      clone = clones_page(b, rc) ? 1 : 0;
      // more writers than references, or holders of one page at two lengths
      if (h_members[e] > rc || h_min[e] != h_max[e]) s_bad_table = 1;
    }
    return AppendSums{n, (len + (long long)n + kPageSize - 1) / kPageSize -
                             (len + kPageSize - 1) / kPageSize + clone, clone};
  };
  AppendSums mine = {0, 0, 0};
  if (!bad)
    for (int b = b0; b < b1; ++b) mine = append_add(mine, one(b));
  AppendSums scan = mine;  // inclusive
  const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const AppendSums up = append_shfl_up(scan, d);
    if (lane >= d) scan = append_add(scan, up);
  }
  if (lane == 31) s_warp[warp] = scan;
  __syncthreads();
  AppendSums before = {0, 0, 0}, total = {0, 0, 0};
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before = append_add(before, s_warp[w]);
    total = append_add(total, s_warp[w]);
  }
  before = append_add(before, scan);  // up to and including this thread's run
  before.tokens -= mine.tokens;
  before.pops -= mine.pops;
  before.clones -= mine.clones;
  if (tid == 0) {
    const bool free_ok = s_free >= 0 && s_free <= p.physical_pages;
    s_status = s_bad_count || total.tokens > p.max_tokens ? kAppendBadCount
               : s_bad_table || !free_ok                  ? kAppendBadTable
               : total.pops > s_free                      ? kAppendExhausted
                                                          : kAppendOk;
  }
  __syncthreads();
  if (s_status == kAppendOk) {  // the pages to be popped are pages
    bool out = false;
    for (int i = tid; i < int(total.pops); i += kPlanThreads) {
      const int page = p.free_stack_in[s_free - 1 - i];
      out |= page < 0 || page >= p.physical_pages;
    }
    if (__syncthreads_or(out) && tid == 0) s_status = kAppendBadTable;
    __syncthreads();
  }
  const bool ok = s_status == kAppendOk;
  for (int b = b0; b < b1; ++b) {
    const int len = p.lengths_in[b];
    if (!ok) {
      p.query_start[b] = 0;
      p.lengths_out[b] = len;
      p.scratch[b] = -1;
      continue;
    }
    const AppendSums s = one(b);
    p.query_start[b] = int(before.tokens);
    p.scratch[b] = int(before.pops) * 2 + s.clones;
    if (s.clones) {
      p.clones[before.clones] = h_page[entry[b]];
      p.clones[p.batch + before.clones] = p.free_stack_in[s_free - 1 - int(before.pops)];
      p.clones[2 * p.batch + before.clones] = len % kPageSize;
    }
    p.lengths_out[b] = len + int(s.tokens);
    before = append_add(before, s);
  }
  const int nclones = ok ? total.clones : 0;
  for (int i = nclones + tid; i < p.batch; i += kPlanThreads)
    p.clones[i] = p.clones[p.batch + i] = p.clones[2 * p.batch + i] = -1;
  if (tid == 0) {
    p.query_start[p.batch] = ok ? int(total.tokens) : 0;
    p.scratch[p.batch] = s_free;
    *p.free_count = ok ? s_free - int(total.pops) : s_free;
    p.counts[0] = ok ? int(total.tokens) : 0;
    p.counts[1] = nclones;
    p.counts[2] = s_status;
  }
}

// The plan written out: blocks [0, row_blocks) take a page table row a warp,
// the others kExpandTokens tokens each.
__global__ void __launch_bounds__(kExpandThreads)
    append_expand_kernel(const AppendPlanParams p, int row_blocks) {
  const int tid = threadIdx.x, lane = tid & 31;
  grid_launch_dependents();
  grid_dependency_wait();
  const int top = p.scratch[p.batch] - 1;  // the stack's top before the pops
  if (int(blockIdx.x) < row_blocks) {
    const int b = blockIdx.x * (kExpandThreads / 32) + (tid >> 5);
    if (b >= p.batch) return;
    const int* in = p.pages_in + size_t(b) * p.max_pages_in;
    int* out = p.pages_out + size_t(b) * p.max_pages_out;
    const bool in_place = p.pages_in == p.pages_out;
    if (p.scratch[b] < 0) {  // no plan: the row as it was, the whole of it at a malformed length
      const int len = p.lengths_out[b];
      const int have = len < 0 || len > p.max_pages_in * kPageSize ? p.max_pages_in
                                                                   : (len + kPageSize - 1) / kPageSize;
      for (int c = lane; c < p.max_pages_out && !in_place; c += 32) out[c] = c < have ? in[c] : -1;
      return;
    }
    const int n = p.query_start[b + 1] - p.query_start[b], len = p.lengths_out[b] - n;
    const int have = (len + kPageSize - 1) / kPageSize;  // (<= max_pages_in)
    const int want = (len + n + kPageSize - 1) / kPageSize;
    const int pop = p.scratch[b] >> 1, clone = p.scratch[b] & 1;
    const int first = in_place ? have - clone : 0, end = in_place ? want : p.max_pages_out;
    for (int c = first + lane; c < end; c += 32) {
      int page = -1;
      if (c < have - clone || (c < have && !clone)) {
        page = in[c];
      } else if (c < want) {
        if (c < have) atomicSub(&p.refcount[in[c]], 1);  // the cloned page's reference
        page = p.free_stack_in[top - (pop + c - (have - clone))];
        p.refcount[page] = 1;
      }
      out[c] = page;
    }
    return;
  }
  const int t0 = (int(blockIdx.x) - row_blocks) * kExpandTokens;
  const int total = p.query_start[p.batch];
  for (int t = t0 + tid; t < min(t0 + kExpandTokens, p.max_tokens); t += kExpandThreads) {
    int slot = -1, pos = -1;
    if (t < total) {
      int lo = 0, hi = p.batch;  // the sequence: the last whose start is at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.query_start[mid] <= t) lo = mid; else hi = mid;
      }
      const int start = p.query_start[lo], n = p.query_start[lo + 1] - start;
      const int len = p.lengths_out[lo] - n;
      const int have = (len + kPageSize - 1) / kPageSize;
      const int pop = p.scratch[lo] >> 1, clone = p.scratch[lo] & 1;
      pos = len + (t - start);
      const int c = pos / kPageSize;
      // (a row's last page is only replaced when it is cloned: never read here then)
      const int page = c < have - clone ? p.pages_in[size_t(lo) * p.max_pages_in + c]
                                        : p.free_stack_in[top - (pop + c - (have - clone))];
      slot = page * kPageSize + pos % kPageSize;
    }
    p.slot_map[t] = slot;
    p.positions[t] = pos;
  }
}

struct AppendKvParams {
  int tokens, row_vecs, head_vecs;  // 16-byte pieces of a token's row and of one head
  int physical_pages, max_clones;
  const uint4* k;
  const uint4* v;
  long long k_stride, v_stride;  // 16-byte pieces between tokens
  uint4* cache_k;
  uint4* cache_v;
  long long block_stride, slot_stride, head_stride;  // in 16-byte pieces
  const int* slot_map;
  const int* clones;  // [3, max_clones] or null
  const int* counts;  // [1]: the number of clones, or null with clones null
  unsigned* err;
};

constexpr int kAppendThreads = 256;
constexpr int kAppendVecs = 4;

// Blocks [0, token_blocks) copy rows, K (blockIdx.y 0) or V (1); block
// token_blocks + c copies clone c's valid slots. A clone reads slots below its
// sequence's length and every row goes to a slot at or past one, so neither
// waits for the other.
__global__ void __launch_bounds__(kAppendThreads)
    append_kv_kernel(const AppendKvParams p, int token_blocks, int tokens_per_block) {
  grid_launch_dependents();
  grid_dependency_wait();
  const bool is_v = blockIdx.y != 0;
  uint4* cache = is_v ? p.cache_v : p.cache_k;
  if (int(blockIdx.x) >= token_blocks) {
    const int c = int(blockIdx.x) - token_blocks;
    if (c >= min(max(*p.counts, 0), p.max_clones)) return;
    const int src = p.clones[c], dst = p.clones[p.max_clones + c];
    const int slots = p.clones[2 * p.max_clones + c];
    if (src < 0 || src >= p.physical_pages || dst < 0 || dst >= p.physical_pages || src == dst ||
        slots < 0 || slots > kPageSize) {
      if (threadIdx.x == 0) atomicOr(p.err, kErrCommitIndex);
      return;
    }
    for (int i = threadIdx.x; i < slots * p.row_vecs; i += kAppendThreads) {
      const int s = i / p.row_vecs, r = i % p.row_vecs;
      const long long at = s * p.slot_stride + (r / p.head_vecs) * p.head_stride + r % p.head_vecs;
      cache[dst * p.block_stride + at] = cache[src * p.block_stride + at];
    }
    return;
  }
  const uint4* x = is_v ? p.v : p.k;
  const long long xs = is_v ? p.v_stride : p.k_stride;
  const int t0 = int(blockIdx.x) * tokens_per_block;
  const int nt = min(tokens_per_block, p.tokens - t0);
  // kAppendVecs pieces of a thread in flight before the first is stored (the
  // stores could be the next loads' sources for all the compiler knows): 18k rows of
  // 2 KB went from 5.54 to 5.71 TB/s.
  for (int i0 = threadIdx.x; i0 < nt * p.row_vecs; i0 += kAppendVecs * kAppendThreads) {
    uint4 val[kAppendVecs];
    long long to[kAppendVecs];
#pragma unroll
    for (int j = 0; j < kAppendVecs; ++j) {
      const int i = i0 + j * kAppendThreads;
      to[j] = -1;
      if (i >= nt * p.row_vecs) continue;
      const int t = t0 + i / p.row_vecs, r = i % p.row_vecs;
      const int slot = p.slot_map[t];
      if (slot < 0 || slot >= p.physical_pages * kPageSize) {
        if (slot != -1 && r == 0) atomicOr(p.err, kErrCommitIndex);
        continue;
      }
      val[j] = __ldcs(x + t * xs + r);
      to[j] = (slot / kPageSize) * p.block_stride + (slot % kPageSize) * p.slot_stride +
              (r / p.head_vecs) * p.head_stride + r % p.head_vecs;
    }
#pragma unroll
    for (int j = 0; j < kAppendVecs; ++j)
      if (to[j] >= 0) cache[to[j]] = val[j];
  }
}

}  // namespace bc
