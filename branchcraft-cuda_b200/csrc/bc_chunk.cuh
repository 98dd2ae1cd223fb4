// Attention of a chunk of new tokens over the paged cache, on the 5th-generation
// tensor cores. Query row (token t of request b, head h) at position
// p = length_b - n_b + i (i: the token's place among the request's n_b) sees the
// keys lo <= j < hi,
//   hi = max(p + 1, prefix_b), lo = max(0, p + 1 - window, key_start_t),
// with scores x_j = scale q.k_j, capped to softcap tanh(x_j / softcap), less
// slope_h |p - j|; the output is sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),
// zeros where no key is seen. Scores that are not finite go through this formula
// as they are: a row that sees +inf or NaN, or nothing but -inf, is NaN.
//
// Work. A row tile is up to 128 (token, query head of one KV head) pairs, so a
// K/V tile read once serves the whole group; an item is one block of two row
// tiles of one request and KV head against the keys its rows see, in tiles of
// 128 keys. Blocks with more than 128 rows are DUAL: softmax group g owns row
// tile g and every key tile serves both. Smaller ones (a decode step: the group's
// heads of one token) are ALT: both groups have the same rows and take alternate
// key tiles, merged at the item's end.
//
// Schedule. One block per SM; the key tiles of all items, laid end to end, are
// cut into equal shares, computed from the lengths on the device by every block
// alike (no host round trip, no counters). A cut inside an item leaves FP32
// partial states (m, l, O) that chunk_merge_kernel joins in order, so results do
// not depend on timing.
//
// Warps: 0-3 and 4-7 softmax groups 0 and 1 (thread = row = TMEM lane), 8 the
// scheduler (item descriptors, Q) and V producer, 10 the K producer (a ring each,
// eight 16-row boxes a tile), 9 the issuer of S = Q K^T, 11 of O += P V. TMEM holds one S (128
// columns) that the groups use in turn, P of each group (64, 16-bit pairs) and O of
// each (128). A group keeps S only while it loads its scores into registers, so the
// next S, of the other group, is computed beside its exponentials, and a group's own
// next scores wait for it when it is done. (With a P over each group's own S, S had
// to wait for the softmax and P V: 3800 cycles a key tile and pair of row tiles, the
// softmaxes and products in turns; their sums are 2048 each.)
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "bc_attn.cuh"

namespace bc {

constexpr int kChThreads = 384;
constexpr int kChMergeThreads = 256;
constexpr int kChTile = 128;      // keys of a tile: eight pages
constexpr int kChDescs = 4;       // item descriptors in flight
constexpr int kChMaxBatch = 4096;
constexpr int kChWhole = 5;       // key tiles of an item that is never split
// What the shares balance, in the time of an ALT key tile: a DUAL tile is two, and
// an item costs this much beside its tiles (its Q, its first scores, its epilogue).
constexpr int kChItemCost = 5;
// Registers: launched at 168 a thread (65,536 / 384, in eights); the softmax
// groups grow to 208 (a row's 128 scores stay in registers), the others shrink
// to 88: together the launch's total.
constexpr int kChLaunchRegs = 168, kChSoftmaxRegs = 208, kChOtherRegs = 88;
static_assert(256 * kChSoftmaxRegs + 128 * kChOtherRegs == kChThreads * kChLaunchRegs,
              "the register split must use exactly the launch budget");

// softcap tanh(x scale / softcap) of a score x, in log2 units: with x' = x pre, x' times a
// polynomial of x'^2 while |x'| < near, else by its exponential. pre is 1 where the
// coefficients, whose last holds the eighth power of scale / softcap, are ordinary
// numbers; elsewhere it is scale / softcap itself, for one multiplication more.
struct ChunkCap {
  float k[5];
  float near, arg, log2, pre;
};

struct ChunkParams {
  int batch, tokens, hq, hkv, group;
  int tile_tokens;            // tokens of a row tile: 128 / group
  int max_pages, physical_pages;
  int window;                 // 0: none
  int head_blocks;            // head stride in 64-element blocks
  const int* pages;           // [batch, max_pages]
  const int* query_start;     // [batch + 1]
  const int* lengths;         // [batch]
  const int* prefix;          // [batch] or null
  const int* key_start;       // [tokens] or null
  const float* slopes;        // [hq] or null
  void* out;                  // [tokens, hq, D]
  int out_f32;
  float scale_log2;           // scale * log2(e)
  ChunkCap cap;               // (used with a cap)
  // workspace of split items (null when none can be split)
  float4* part_o;             // [blocks * 2][D / 4][part_rows]
  float2* part_ml;            // [blocks * 2][part_rows]
  int* sched;                 // [blocks][8]
  int part_rows;
  unsigned smem_bytes;        // dynamic shared memory of the launch
  unsigned* err;
  unsigned token;
};

// A request's rows and keys, with malformed values brought into range.
struct ChunkRequest {
  int first, n, len, prefix;  // first token, tokens, keys, keys open to all
};
__device__ __forceinline__ ChunkRequest chunk_request(const ChunkParams& p, int b) {
  const int a = p.query_start[b], e = p.query_start[b + 1], len = p.lengths[b];
  const int pre = p.prefix ? p.prefix[b] : 0;
  ChunkRequest r;
  r.first = min(max(a, 0), p.tokens);
  r.n = max(min(e, p.tokens) - r.first, 0);
  r.len = min(max(len, 0), p.max_pages * kPageSize);
  r.prefix = min(max(pre, 0), r.len);
  if (a != r.first || e != r.first + r.n || len != r.len || r.len < r.n) atomicOr(p.err, kErrLength);
  return r;
}

// The keys that some row of a block of `cnt` tokens from the request's token
// `i0` on may see, and their tiles (at least one: a block without keys still
// writes its zeros).
struct ChunkRange {
  int lo, hi, t0, tiles;
};
__device__ __forceinline__ ChunkRange chunk_range(const ChunkParams& p, const ChunkRequest& r,
                                                  int i0, int cnt) {
  const int pos = r.len - r.n + i0;
  ChunkRange g;
  g.hi = max(max(pos + cnt, r.prefix), 0);
  g.lo = p.window ? int(max((long long)pos + 1 - p.window, 0ll)) : 0;
  if (p.key_start) {
    int ks = 0x7fffffff;
    for (int i = 0; i < cnt; ++i) ks = min(ks, p.key_start[r.first + i0 + i]);
    g.lo = max(g.lo, ks);
  }
  g.lo = min(g.lo, g.hi);
  g.t0 = g.lo / kChTile;
  g.tiles = max((g.hi + kChTile - 1) / kChTile - g.t0, 1);
  return g;
}

// A block's share of the work: its number of key tiles times this, and kChItemCost.
__device__ __forceinline__ int chunk_weight(const ChunkParams& p, int cnt) {
  return cnt > p.tile_tokens ? 2 : 1;
}
__device__ __forceinline__ int chunk_cost(const ChunkParams& p, const ChunkRequest& r, int blk) {
  const int i0 = blk * 2 * p.tile_tokens, cnt = min(2 * p.tile_tokens, r.n - i0);
  return kChItemCost + chunk_weight(p, cnt) * chunk_range(p, r, i0, cnt).tiles;
}

// One piece of an item, as every role reads it.
struct ChunkDesc {
  int first, ntok;       // the block's first token (row of q) and its tokens
  int pos;               // position of the first
  int prefix, lo, hi;    // keys open to all, and the block's range
  int request, head;
  int t0, nt;            // first key tile and number of tiles of this piece
  int dual;              // two row tiles
  int slot;              // partial state's place, or -1: the whole item
  int end;               // no item: the last descriptor
};

template <int D>
struct ChunkGeom {
  static constexpr int KB = D / 64;
  static constexpr int kRowTile = 128 * D * 2;   // Q of a row tile, K or V of a key tile
  static constexpr int kPageBytes = 16 * D * 2;
  static constexpr int kGroupBytes = KB * 1024;  // eight keys
  // rings: S = Q K^T runs up to a tile ahead of O += P V and frees K first
  static constexpr int kKStages = D == 128 ? 3 : 4, kVStages = D == 128 ? 2 : 4;
  static constexpr int kStages = kKStages + kVStages;
  // barriers and small state lie before the 1024-byte aligned tiles
  static constexpr int kBars = 2 * kStages + 3 + 14 + 2 * kChDescs;
  static constexpr int kMiscBytes = kBars * 8 + 16 + kChDescs * int(sizeof(ChunkDesc));
  static constexpr int kQOff = 0;
  static constexpr int kRingOff = 2 * kRowTile;
  static constexpr int kMlOff = kRingOff + kStages * kRowTile;  // [2][128] (m, l)
  static constexpr int kTileBytes = kMlOff + 2 * 128 * 8;
  static_assert(kMiscBytes <= 1008, "the small state fits before the first tile");
  static_assert(kChMaxBatch * 24 <= kStages * kRowTile, "the plan's requests fit in the ring");
  // with `fixed` bytes of static shared memory before the dynamic part
  static size_t smem_bytes(size_t fixed) {
    const size_t at = (fixed + 15) / 16 * 16;
    return (at + kMiscBytes + 1023) / 1024 * 1024 - at + kTileBytes;
  }
  // TMEM columns: S, P of group g, O of group g
  static constexpr uint32_t kTmemP = 128, kTmemO = 256, kTmemCols = 512;
};

// 5-D tiled load: one page's 16 rows of one head as [2][KB][8][128 bytes], so
// that consecutive pages continue the same row of 8-key groups.
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2, int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3), "r"(c4)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// Waits out copies in flight on a failing launch: as mbar_wait, but deaf to the
// launch's abort mark (at most 10 ms).
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  const unsigned long long start = globaltimer_ns();
  while (!mbar_try_wait(bar, parity) && globaltimer_ns() - start < 10000000ull) {
  }
}

__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value)
    return unpack_half2(w);
  else
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 32 lanes x 8 columns of tensor memory, as tmem_ld32 and its companions.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_bind8(uint32_t (&r)[8]) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                    "+r"(r[6]), "+r"(r[7]));
}

// Two FP32 lanes in one instruction: (a0, a1) * (b, b) + (c, c).
__device__ __forceinline__ void fma_pair(float a0, float a1, float b, float c, float& d0,
                                         float& d1) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void add_pair(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}

// Largest magnitude of three.
__device__ __forceinline__ float fmax3_abs(float a, float b, float c) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 32 bytes at once (the address a multiple of 32).
__device__ __forceinline__ void st_global_v8(void* to, uint32_t a, uint32_t b, uint32_t c,
                                             uint32_t d, uint32_t e, uint32_t f, uint32_t g,
                                             uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(a), "r"(b),
               "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h)
               : "memory");
}

// MOD: bit 0 the tanh cap, bit 1 the distance bias. F32: FP32 output, whose
// probabilities are held as two 16-bit numbers, handed over and multiplied one after
// the other (P has no second place in TMEM).
template <int D, typename T, int MOD, bool F32>
__global__ void __launch_bounds__(kChThreads, 1)
    chunk_mma_kernel(const __grid_constant__ ChunkParams p, const __grid_constant__ CUtensorMap qmap,
                     const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap) {
  using G = ChunkGeom<D>;
  constexpr int KB = G::KB, NK = G::kKStages, NV = G::kVStages;
  constexpr int kParts = F32 ? 2 : 1;  // of P
  constexpr float kNegInf = -INFINITY, kLowest = -3.402823466e38f;
  constexpr uint32_t kBf16 = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
  constexpr uint32_t kIdescS = umma_idesc_f16(128, kChTile, false, false) | kBf16;
  constexpr uint32_t kIdescPV = umma_idesc_f16(128, D, false, true) | kBf16;

  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + G::kMiscBytes + 1023) & ~uintptr_t(1023));
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem_raw);  // [NK] a K tile landed
  uint64_t* k_empty = k_full + NK;      // [NK] its S products are done
  uint64_t* v_full = k_empty + NK;      // [NV]
  uint64_t* v_empty = v_full + NV;      // [NV] its P V products are done
  uint64_t* q_full = v_empty + NV;
  uint64_t* q_free = q_full + 1;        // the item's S products are done
  uint64_t* s_free = q_free + 1;        // S is in its group's registers (4 warps)
  uint64_t* s_full = s_free + 1;        // [2] S holds scores of group g
  uint64_t* p_half = s_full + 2;        // [2] P of group g written: the first 64 keys (4 warps)
  uint64_t* p_full = p_half + 2;        // [2] and the others
  uint64_t* p_done = p_full + 2;        // [2] its product is complete: P free, O up to date
  uint64_t* xch = p_done + 2;           // [2] ALT: group g's (m, l) written (4 warps)
  uint64_t* xch_done = xch + 2;         // [2] ALT: group g has read both O (4 warps)
  uint64_t* fin = xch_done + 2;         // [2] an issuer's last product
  uint64_t* desc_full = fin + 2;        // [kChDescs]
  uint64_t* desc_empty = desc_full + kChDescs;  // [kChDescs] read by 11 warps
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(desc_empty + kChDescs);
  ChunkDesc* descs = reinterpret_cast<ChunkDesc*>(reinterpret_cast<uint8_t*>(desc_empty + kChDescs) + 16);
  float2* ml_x = reinterpret_cast<float2*>(tiles + G::kMlOff);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (uint32_t(tiles - smem_raw) + G::kTileBytes > p.smem_bytes) {  // (never: the host's sum)
    if (tid == 0) atomicOr(p.err, kErrTimeout);
    return;
  }
  if (tid == 0) {
    s_launch_token = p.token;
    for (int s = 0; s < NK; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < NV; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(s_free, 4);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_half[g], 4);
      mbar_init(&p_full[g], 4);
      mbar_init(&p_done[g], 1);
      mbar_init(&xch[g], 4);
      mbar_init(&xch_done[g], 4);
      mbar_init(&fin[g], 1);
    }
    for (int s = 0; s < kChDescs; ++s) {
      mbar_init(&desc_full[s], 1);
      mbar_init(&desc_empty[s], 11);
    }
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, G::kTmemCols);
    tmem_relinquish();
    tc_fence_before();
  }
  if (warp == 8 && lane < 3) prefetch_tmap(lane == 0 ? &qmap : lane == 1 ? &kmap : &vmap);
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  grid_launch_dependents();  // (TMEM is allocated: a waiting successor cannot hold it back)
  grid_dependency_wait();

  // ---- plan: every request and its cost (per KV head), into the idle rings
  const int block_tokens = 2 * p.tile_tokens;
  long long* cost_of = reinterpret_cast<long long*>(tiles + G::kRingOff);
  ChunkRequest* request_of = reinterpret_cast<ChunkRequest*>(cost_of + kChMaxBatch);
  for (int base = warp * 32; base < p.batch; base += (kChThreads / 32) * 32) {
    const int b = base + lane;
    ChunkRequest r = {0, 0, 0, 0};
    if (b < p.batch) r = chunk_request(p, b);
    const int nblk = (r.n + block_tokens - 1) / block_tokens;
    long long sum = 0;
    if (nblk <= 4)
      for (int j = 0; j < nblk; ++j) sum += chunk_cost(p, r, j);
    for (unsigned many = __ballot_sync(0xffffffffu, nblk > 4); many; many &= many - 1) {
      const int src = __ffs(many) - 1;  // a long chunk: its blocks spread over the warp
      const ChunkRequest o = {__shfl_sync(0xffffffffu, r.first, src),
                              __shfl_sync(0xffffffffu, r.n, src),
                              __shfl_sync(0xffffffffu, r.len, src),
                              __shfl_sync(0xffffffffu, r.prefix, src)};
      long long part = 0;
      for (int j = lane; j * block_tokens < o.n; j += 32) part += chunk_cost(p, o, j);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
      if (lane == src) sum = part;
    }
    if (b < p.batch) {
      cost_of[b] = sum;
      request_of[b] = r;
    }
  }
  fence_proxy_async_smem();  // (copies will follow into the same memory)
  __syncthreads();

  const uint32_t lane_addr = uint32_t((warp & 3) * 32) << 16;
  bool ok = true;
  if (warp >= 8) {
    regs_decrease<kChOtherRegs>();
    // The copies of an item's K (or V) tiles, the warp's `tile0`-th on: lane l holds
    // the page id of page (l & 7) of tile 4 batch + l / 8, loaded a batch ahead, and
    // eight lanes issue a box each (a warp issues one per 70 ns or so: a producer
    // each for K and V, since one for both spent 1090 cycles a tile load: 111 -> 104 us).
    auto copy_tiles = [&](auto is_v, const ChunkDesc& d, unsigned tile0, unsigned& issued) -> bool {
      constexpr bool V = decltype(is_v)::value;
      constexpr int N = V ? NV : NK;
      uint64_t *full = V ? v_full : k_full, *empty = V ? v_empty : k_empty;
      const int* row = p.pages + size_t(d.request) * p.max_pages;
      auto load_id = [&](int first) -> int {
        const int j = first + (lane >> 3);
        const int pg = (d.t0 + j) * (kChTile / kPageSize) + (lane & 7);
        // pages that no row of the block sees stay out: the copy fills zeros
        if (j >= d.nt || pg * kPageSize >= d.hi || (pg + 1) * kPageSize <= d.lo) return -1;
        const int id = __ldg(row + pg);
        if (id >= 0 && id < p.physical_pages) return id;
        atomicOr(p.err, kErrPageRange);
        return -1;
      };
      int cur = load_id(0), nxt = load_id(4);
      for (int j = 0; j < d.nt; ++j) {
        if (j > 0 && (j & 3) == 0) {
          cur = nxt;
          nxt = load_id(j + 4);
        }
        const unsigned s = tile0 + unsigned(j);
        const int st = int(s % N);
        if (s >= N && !__all_sync(0xffffffffu, mbar_wait(&empty[st], ((s / N) - 1) & 1))) return false;
        if (lane == 0) mbar_arrive_expect_tx(&full[st], uint32_t(G::kRowTile));
        const int id = __shfl_sync(0xffffffffu, cur, (j & 3) * 8 + (lane & 7));
        if (lane < 8)
          tma_load_5d(tiles + G::kRingOff + ((V ? NK : 0) + st) * G::kRowTile + lane * G::kPageBytes,
                      V ? &vmap : &kmap, &full[st], 0, 0, d.head * p.head_blocks, 0, id);
        __syncwarp();
        issued = s + 1;
      }
      return true;
    };
    // A failing launch waits out the copies in flight: the ring's last tiles.
    auto drain_tiles = [&](auto is_v, unsigned issued) {
      constexpr bool V = decltype(is_v)::value;
      constexpr unsigned N = V ? NV : NK;
      uint64_t* full = V ? v_full : k_full;
      if (lane == 0)
        for (unsigned s = issued - min(issued, N); s < issued; ++s)
          mbar_drain(&full[s % N], (s / N) & 1);
      __syncwarp();
    };
    if (warp == 8) {
      // ------------------------------------------- scheduler and V producer
      // This block's share: from its own cut (found by lanes 0-15) up to the next
      // block's (lanes 16-31). Cuts inside an item fall on multiples of `grain`
      // tiles from its start (a thirty-second of a share, at least 2, which bounds what
      // rounding adds to a block) or on its ends; an item of no more than kChWhole
      // tiles has no cut.
      const int half = lane >> 4, hl = lane & 15;
      const int per_lane = (p.batch + 15) / 16;
      const int sb0 = min(p.batch, hl * per_lane), sb1 = min(p.batch, sb0 + per_lane);
      auto scan = [&](long long v) {  // inclusive, over the lanes of a half
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
          const long long up = __shfl_up_sync(0xffffffffu, v, d, 16);
          if (hl >= d) v += up;
        }
        return v;
      };
      // the half's last lane whose run (of cost `mine` per head, after `pre`) begins
      // at or before u
      auto owner = [&](long long mine, long long pre, long long u) -> int {
        const unsigned at =
            (__ballot_sync(0xffffffffu, mine > 0 && pre * p.hkv <= u) >> (16 * half)) & 0xffffu;
        return at ? 31 - __clz(at) : 0;
      };
      long long mine = 0;
      for (int b = sb0; b < sb1; ++b) mine += cost_of[b];
      long long incl = scan(mine);
      const long long cost = __shfl_sync(0xffffffffu, incl, 15, 16) * p.hkv;  // of the whole call
      const long long u = (long long)(double(cost) * double(blockIdx.x + half) / double(gridDim.x));
      const bool in = u < cost;  // (else the call's end: request p.batch)
      // the request
      int req = p.batch, blk = 0, head = 0, off = 0;
      long long at = incl - mine;
      int src = owner(mine, at, u);
      if (in && hl == src)
        for (req = sb0; (at + cost_of[req]) * p.hkv <= u; ++req) at += cost_of[req];
      req = __shfl_sync(0xffffffffu, req, src, 16);
      long long rem = u - __shfl_sync(0xffffffffu, at, src, 16) * p.hkv;
      ChunkRequest r = {0, 0, 0, 0};
      if (in) r = request_of[req];
      // its block, a run of consecutive ones a lane
      const int nblk = (r.n + block_tokens - 1) / block_tokens;
      const int run = (nblk + 15) / 16, j0 = min(nblk, hl * run), j1 = min(nblk, j0 + run);
      mine = 0;
      for (int j = j0; j < j1; ++j) mine += chunk_cost(p, r, j);
      incl = scan(mine);
      at = incl - mine;
      src = owner(mine, at, rem);
      int n = 1;
      if (in && hl == src)
        for (blk = j0; n = chunk_cost(p, r, blk), (at + n) * p.hkv <= rem; ++blk) at += n;
      blk = __shfl_sync(0xffffffffu, blk, src, 16);
      n = __shfl_sync(0xffffffffu, n, src, 16);
      rem -= __shfl_sync(0xffffffffu, at, src, 16) * p.hkv;
      // its head and tile
      const int weight = chunk_weight(p, r.n - blk * block_tokens);
      const int grain = max(2, int(fminf(float(cost) / float(gridDim.x * 32 * weight), 1048576.f)));
      if (in) {
        head = int(float(rem) / float(n));  // (rem < n * hkv; put right below)
        while ((long long)head * n > rem) --head;
        while ((long long)(head + 1) * n <= rem) ++head;
        off = max(int(rem - (long long)head * n) - kChItemCost, 0) >> (weight - 1);
        n = (n - kChItemCost) >> (weight - 1);
        off = n <= kChWhole ? (2 * off > n ? n : 0) : (off + grain / 2) / grain * grain;
        if (off > 0 && n - off < (grain + 1) / 2) {  // the next item's start
          off = 0;
          if (++head == p.hkv) {
            head = 0;
            if (++blk == nblk) {
              blk = 0;
              do {
                ++req;
              } while (req < p.batch && request_of[req].n == 0);
              if (req < p.batch) r = request_of[req];
            }
          }
        }
      }
      const int e_req = __shfl_sync(0xffffffffu, req, 16), e_blk = __shfl_sync(0xffffffffu, blk, 16),
                e_head = __shfl_sync(0xffffffffu, head, 16), e_off = __shfl_sync(0xffffffffu, off, 16);
      req = __shfl_sync(0xffffffffu, req, 0);
      blk = __shfl_sync(0xffffffffu, blk, 0);
      head = __shfl_sync(0xffffffffu, head, 0);
      off = __shfl_sync(0xffffffffu, off, 0);
      r.first = __shfl_sync(0xffffffffu, r.first, 0);
      r.n = __shfl_sync(0xffffffffu, r.n, 0);
      r.len = __shfl_sync(0xffffffffu, r.len, 0);
      r.prefix = __shfl_sync(0xffffffffu, r.prefix, 0);
      ChunkRange g = {0, 0, 0, 1};
      auto load_block = [&] {  // the current block's range
        g = chunk_range(p, r, blk * block_tokens, min(block_tokens, r.n - blk * block_tokens));
      };
      if (req < p.batch) load_block();
      auto next_item = [&] {
        off = 0;
        if (++head < p.hkv) return;
        head = 0;
        if ((++blk) * block_tokens >= r.n) {
          blk = 0;
          // the next request with tokens (the plan is gone: the rings are in use),
          // 32 looked at together
          for (++req; req < p.batch; req += 32) {
            const int b = req + lane;
            const bool some = b < p.batch && chunk_request(p, b).n > 0;
            const unsigned with = __ballot_sync(0xffffffffu, some);
            if (with) {
              req += __ffs(with) - 1;
              break;
            }
          }
          req = min(req, p.batch);
          if (req < p.batch) r = chunk_request(p, req);
        }
        if (req < p.batch) load_block();
      };
      // tiles of the current item that are this block's, from `off` on
      auto mine_here = [&]() -> int {
        if (req >= p.batch) return 0;
        return (req == e_req && blk == e_blk && head == e_head ? e_off : g.tiles) - off;
      };
      int left = mine_here();
      // for the merge: the first piece continues an item that goes on (1) or ends
      // (2) here, or this block has no share (3); and the item that starts here
      // and goes on
      int cont = left > 0 ? 0 : 3, has = 0, h_first = 0, h_ntok = 0, h_head = 0;
      // The piece at hand as a descriptor, handed to the other warps.
      auto publish = [&](int k) -> ChunkDesc {
        ChunkDesc d = {};
        d.end = left <= 0;
        if (!d.end) {
          const int i0 = blk * block_tokens;
          d.first = r.first + i0;
          d.ntok = min(block_tokens, r.n - i0);
          d.pos = r.len - r.n + i0;
          d.prefix = r.prefix;
          d.lo = g.lo;
          d.hi = g.hi;
          d.request = req;
          d.head = head;
          d.t0 = g.t0 + off;
          d.nt = left;
          d.dual = d.ntok > p.tile_tokens;
          const bool whole = off == 0 && d.nt == g.tiles;
          d.slot = whole ? -1 : int(blockIdx.x) * 2 + (off == 0 ? 1 : 0);
          if (!whole && off == 0) {
            has = 1;
            h_first = d.first;
            h_ntok = d.ntok;
            h_head = head;
          }
          if (off > 0) cont = off + d.nt == g.tiles ? 2 : 1;
        }
        const int ds = k % kChDescs;
        if (k >= kChDescs)
          ok = __all_sync(0xffffffffu, mbar_wait(&desc_empty[ds], ((k / kChDescs) - 1) & 1));
        if (ok && lane == 0) {
          descs[ds] = d;
          mbar_arrive(&desc_full[ds]);
        }
        __syncwarp();
        return d;
      };
      ChunkDesc d = publish(0);
      unsigned tile0 = 0, issued = 0;
      int nq_loaded = 0;  // items whose Q has been asked for
      for (int k = 0; ok && !d.end; ++k) {
        if (k > 0) ok = __all_sync(0xffffffffu, mbar_wait(q_free, (k - 1) & 1));
        if (!ok) break;
        // Q of the block's row tiles; rows past the request's are other tokens'
        // (or zeros past the last): computed, never stored.
        const int nq = d.dual ? 2 : 1;
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full, uint32_t(nq * KB * p.tile_tokens * p.group * 128));
          for (int i = 0; i < nq; ++i)
            for (int kb = 0; kb < KB; ++kb)
              tma_load_3d(tiles + G::kQOff + i * G::kRowTile + kb * (128 * 128), &qmap, q_full,
                          kb * 64, d.head * p.group, d.first + i * p.tile_tokens);
        }
        __syncwarp();
        nq_loaded = k + 1;
        // the next piece is known before this one's V: K runs ahead
        if (off + d.nt < g.tiles) {  // the share ends inside this item
          left = 0;
        } else {
          next_item();
          left = mine_here();
        }
        const ChunkDesc next = publish(k + 1);
        if (ok) ok = copy_tiles(std::true_type{}, d, tile0, issued);
        tile0 += unsigned(d.nt);
        d = next;
      }
      if (p.sched && lane == 0) {
        int* s = p.sched + size_t(blockIdx.x) * 8;
        s[0] = cont;
        s[1] = has;
        s[2] = h_first;
        s[3] = h_ntok;
        s[4] = h_head;
      }
      if (!ok) {
        if (nq_loaded > 0) mbar_drain(q_full, (nq_loaded - 1) & 1);
        drain_tiles(std::true_type{}, issued);
      }
    } else if (warp != 10) {
      // ------------------------------------------------------------ issuers
      // Warp 9: S_g = Q_g K^T, warp 11: O_g += P_g V, the groups in turn. (Two
      // issuers, so that one's waits do not hold back the other's products.) Every
      // barrier is waited for phase by phase.
      const bool is_pv = warp == 11;
      const uint64_t qdesc = umma_desc_sw128(smem_u32(tiles + G::kQOff), 16, 1024);
      const uint64_t kdesc = umma_desc_sw128(smem_u32(tiles + G::kRingOff), 16, G::kGroupBytes);
      const uint64_t vdesc = umma_desc_sw128(
          smem_u32(tiles + G::kRingOff + NK * G::kRowTile), 1024, G::kGroupBytes);
      const bool leader = elect_one();  // issues every product and commit
      unsigned tile = 0, count = 0;     // tiles of the ring, products issued
      uint32_t pc[2] = {0u, 0u};        // P tiles taken of each group
      for (int k = 0; ok; ++k) {
        const int ds = k % kChDescs;
        ok = __all_sync(0xffffffffu, mbar_wait(&desc_full[ds], (k / kChDescs) & 1));
        if (!ok) break;
        const int nt = descs[ds].nt, dual = descs[ds].dual, end = descs[ds].end;
        __syncwarp();
        if (lane == 0) mbar_arrive(&desc_empty[ds]);
        if (end) break;
        if (!is_pv) ok = __all_sync(0xffffffffu, mbar_wait(q_full, k & 1));
        if (!ok) break;
        for (int j = 0; j < nt && ok; ++j, ++tile) {
          const int st = int(tile % (is_pv ? NV : NK));
          ok = __all_sync(0xffffffffu, is_pv ? mbar_wait(&v_full[st], (tile / NV) & 1)
                                             : mbar_wait(&k_full[st], (tile / NK) & 1));
          if (!ok) break;
#pragma unroll 1
          for (int g = dual ? 0 : (j & 1); g <= (dual ? 1 : (j & 1)); ++g, ++count) {
            if (is_pv) {
              const uint64_t vd = vdesc + uint64_t((st * G::kRowTile) >> 4);
              const uint32_t acc = (dual ? j : j >> 1) > 0 ? 1u : 0u;
              // (the first half's products run while the second half of P is
              // still being made)
#pragma unroll
              for (int i = 0; i < 2 * kParts; ++i) {
                const int part = i >> 1, h = i & 1;
                const uint32_t par = (g ? pc[1] : pc[0]) & 1;
                if (h) {
                  if (g) ++pc[1]; else ++pc[0];
                }
                ok = __all_sync(0xffffffffu, mbar_wait(h ? &p_full[g] : &p_half[g], par));
                if (!ok) break;
                tc_fence_after();
                if (leader) {
#pragma unroll
                  for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                    umma_f16_ts(tbase + G::kTmemO + g * 128, tbase + G::kTmemP + g * 64 + kk * 8,
                                vd + uint64_t((kk * 2 * G::kGroupBytes) >> 4), kIdescPV,
                                kk > 0 || part > 0 ? 1u : acc);
                  if (h) {
                    umma_commit(&p_done[g]);
                    if (part == kParts - 1 && (!dual || g == 1)) umma_commit(&v_empty[st]);
                  }
                }
                __syncwarp();
              }
              if (!ok) break;
            } else {
              // S is free once the last group holds its scores in registers
              if (count > 0) ok = __all_sync(0xffffffffu, mbar_wait(s_free, (count - 1) & 1));
              if (!ok) break;
              tc_fence_after();
              const uint64_t qd = qdesc + uint64_t((dual ? g * G::kRowTile : 0) >> 4);
              const uint64_t kd = kdesc + uint64_t((st * G::kRowTile) >> 4);
              if (leader) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                  umma_f16(tbase, qd + uint64_t(((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4),
                           kd + uint64_t(((ks >> 2) * 1024 + (ks & 3) * 32) >> 4), kIdescS,
                           ks > 0 ? 1u : 0u);
                umma_commit(&s_full[g]);
                if (!dual || g == 1) {
                  umma_commit(&k_empty[st]);
                  if (j == nt - 1) umma_commit(q_free);
                }
              }
            }
            __syncwarp();
          }
        }
      }
      if (leader) umma_commit(&fin[is_pv]);
      __syncwarp();
      if (lane == 0) mbar_drain(&fin[is_pv], 0);
      __syncwarp();
    } else {
      // --------------------------------------------------------- K producer
      unsigned tile0 = 0, issued = 0;
      for (int k = 0; ok; ++k) {
        const int ds = k % kChDescs;
        ok = __all_sync(0xffffffffu, mbar_wait(&desc_full[ds], (k / kChDescs) & 1));
        if (!ok) break;
        const ChunkDesc d = descs[ds];
        __syncwarp();
        if (lane == 0) mbar_arrive(&desc_empty[ds]);
        if (d.end) break;
        ok = copy_tiles(std::false_type{}, d, tile0, issued);
        tile0 += unsigned(d.nt);
      }
      if (!ok) drain_tiles(std::false_type{}, issued);
    }
    if (!ok && lane == 0) atomicOr(p.err, kErrTimeout);
    tc_fence_before();
    named_barrier_sync(1, kChThreads);  // every TMEM read and product is done
    if (warp == 9) {
      tc_fence_after();
      tmem_dealloc(tbase, G::kTmemCols);
    }
    return;
  }
  // (the softmax path never rejoins the other: each keeps its register budget)
  {
    // --------------------------------------------------------------- softmax
    regs_increase<kChSoftmaxRegs>();
    const int grp = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t tS = tbase + lane_addr;
    const uint32_t tP = tbase + lane_addr + G::kTmemP + uint32_t(grp) * 64;
    const uint32_t tO = tbase + lane_addr + G::kTmemO + uint32_t(grp) * 128;
    const int row_tok = row / p.group, row_head = row % p.group;
    uint32_t sc = 0, alt = 0;  // tiles of this group, ALT items done
    uint32_t pn = 0;           // P handed over, where that is not one a tile
    // The last P handed over has been multiplied: P is free, O holds its product.
    auto p_taken = [&]() -> bool {
      const uint32_t n = F32 ? pn : sc;
      return n == 0 || __all_sync(0xffffffffu, mbar_wait(&p_done[grp], (n - 1) & 1));
    };
    unsigned tile0 = 0;        // the item's first tile in the rings
    for (int k = 0; ok; ++k) {
      const int ds = k % kChDescs;
      ok = __all_sync(0xffffffffu, mbar_wait(&desc_full[ds], (k / kChDescs) & 1));
      if (!ok) break;
      // (held until the item's end: its fields are read where they are needed)
      const volatile ChunkDesc& d = descs[ds];
      if (d.end) break;
      const bool dual = d.dual != 0;
      const int n_mine = dual ? d.nt : (d.nt + 1 - grp) / 2;
      const int tok = (dual ? grp * p.tile_tokens : 0) + row_tok;
      const bool valid = row_tok < p.tile_tokens && tok < d.ntok;
      const int head = d.head * p.group + row_head;
      const int pos = d.pos + tok;
      // the row's keys (a row of nobody keeps all of them, so as not to send its
      // warp down the masked path: its results are dropped)
      int lo = 0, hi = 0x7fffffff;
      if (valid) {
        hi = max(pos + 1, d.prefix);
        if (p.window) lo = int(max((long long)pos + 1 - p.window, 0ll));
        if (p.key_start) lo = max(lo, __ldg(p.key_start + d.first + tok));
      }
      float slope = 0.f;
      if ((MOD & 2) && valid) slope = __ldg(p.slopes + head) * 1.4426950408889634f;
      const bool idle = __all_sync(0xffffffffu, !valid);  // rows of this warp are nobody's
      float m_ref = kNegInf, l_sum = 0.f;
      // Slots outside the block's range may hold anything: their V rows become
      // zeros, so that 0 * V stays 0 (whole pages outside are zeros already).
      // (DUAL: both groups do, each before its own product.)
      auto zero_pads = [&](int j, int k0) -> bool {
        const int z0 = min(max(d.lo - k0, 0), kChTile), z1 = min(max(d.hi - k0, 0), kChTile);
        if (((z0 | z1) & 15) == 0) return true;
        const unsigned vt = tile0 + unsigned(j);
        if (!__all_sync(0xffffffffu, mbar_wait(&v_full[vt % NV], (vt / NV) & 1))) return false;
        const uint32_t vb = smem_u32(tiles + G::kRingOff) + uint32_t(NK + vt % NV) * G::kRowTile;
        const int pad0 = z0 & 15, pad1 = (16 - (z1 & 15)) & 15;
        for (int c = row; c < (pad0 + pad1) * KB * 8; c += 128) {
          const int i = c / (KB * 8), rem = c % (KB * 8);
          const int key = i < pad0 ? z0 - 1 - i : z1 + (i - pad0);
          st_shared_v4(vb + (key >> 3) * G::kGroupBytes + (rem >> 3) * 1024 + (key & 7) * 128 +
                           ((rem & 7) << 4), 0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        return true;
      };
      if (idle) {  // nothing to compute: the barriers alone
        for (int n = 0; n < n_mine && ok; ++n, ++sc) {
          const int j = dual ? n : 2 * n + grp;
          ok = __all_sync(0xffffffffu, mbar_wait(&s_full[grp], sc & 1));
          if (ok && lane == 0) mbar_arrive(s_free);
          ok = ok && p_taken() && zero_pads(j, (d.t0 + j) * kChTile);
          for (int part = 0; part < kParts && ok; ++part, ++pn) {
            if (part > 0) ok = p_taken();
            __syncwarp();
            if (ok && lane == 0) {
              mbar_arrive(&p_half[grp]);
              mbar_arrive(&p_full[grp]);
            }
          }
        }
      }
      for (int n = 0; n < n_mine && !idle; ++n) {
        const int j = dual ? n : 2 * n + grp;
        const int k0 = (d.t0 + j) * kChTile;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[grp], sc & 1));
        if (!ok) break;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, s[c]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_bind32(s[c]);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
        // Scores in log2 units when they are capped or biased; otherwise the
        // scale (> 0) waits for the exponent's multiply-add.
        if constexpr (MOD & 1) {
          // cap * tanh(u), u = x scale / cap, by the score's own size, so that no other
          // score changes a bit of it: below |u| = 0.55, where scores of a model trained
          // with its cap lie, as x Q(x^2), an odd polynomial of u of degree 9 (ChunkCap),
          // 6 operations a score, two scores at a time; beyond as
          // cap - 2 cap / (1 + exp(2 u)), two more results of the exponential unit, which
          // bounds the softmax. A warp without such scores skips that form.
          if (p.cap.pre != 1.f) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                s[c][e] = __float_as_uint(__uint_as_float(s[c][e]) * p.cap.pre);
          }
          float big = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 2)
              big = fmax3_abs(big, __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
          auto both = [](float x) { return pair_of(x, x); };
          const uint64_t k0 = both(p.cap.k[0]), k1 = both(p.cap.k[1]), k2 = both(p.cap.k[2]),
                         k3 = both(p.cap.k[3]), k4 = both(p.cap.k[4]);
          auto near = [&](float x0, float x1) -> float2 {
            const uint64_t x = pair_of(x0, x1), t = mul2(x, x);
            return pair_floats(mul2(x, fma2(t, fma2(t, fma2(t, fma2(t, k4, k3), k2), k1), k0)));
          };
          if (__all_sync(0xffffffffu, big < p.cap.near)) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 y = near(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
                s[c][e] = __float_as_uint(y.x);
                s[c][e + 1] = __float_as_uint(y.y);
              }
          } else {
            auto far = [&](float x) {
              return fmaf(-2.f * p.cap.log2, fast_rcp(1.f + fast_exp2(x * p.cap.arg)), p.cap.log2);
            };
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float x0 = __uint_as_float(s[c][e]), x1 = __uint_as_float(s[c][e + 1]);
                const float2 y = near(x0, x1);
                s[c][e] = __float_as_uint(fabsf(x0) < p.cap.near ? y.x : far(x0));
                s[c][e + 1] = __float_as_uint(fabsf(x1) < p.cap.near ? y.y : far(x1));
              }
            __syncwarp();
          }
        }
        if constexpr (MOD & 2) {
          const float d0 = float(k0 - pos);
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x = __uint_as_float(s[c][e]);
              s[c][e] = __float_as_uint(fmaf(-slope, fabsf(d0 + float(c * 32 + e)),
                                             (MOD & 1) ? x : x * p.scale_log2));
            }
        }
        const int a = lo - k0, b = hi - k0;
        const bool open = __all_sync(0xffffffffu, a <= 0 && b >= kChTile);  // no mask
        if (!open) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int bc = min(max(b - c * 32, 0), 32), ac = min(max(a - c * 32, 0), 32);
            const uint32_t below_b = bc == 32 ? 0xffffffffu : (1u << bc) - 1u;
            const uint32_t below_a = ac == 32 ? 0xffffffffu : (1u << ac) - 1u;
            const uint32_t bits = below_b & ~below_a;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((bits >> e) & 1u)) s[c][e] = __float_as_uint(kNegInf);
          }
        }
        float mx;
        {
          float m8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            m8[i] = fmax3(__uint_as_float(s[0][i]), __uint_as_float(s[0][i + 8]),
                          __uint_as_float(s[0][i + 16]));
            m8[i] = fmax3(m8[i], __uint_as_float(s[0][i + 24]), __uint_as_float(s[1][i]));
#pragma unroll
            for (int q = 1; q < 4; ++q) {
              m8[i] = fmax3(m8[i], __uint_as_float(s[q][i + 8]), __uint_as_float(s[q][i + 16]));
              if (q < 3)
                m8[i] = fmax3(m8[i], __uint_as_float(s[q][i + 24]), __uint_as_float(s[q + 1][i]));
              else
                m8[i] = fmaxf(m8[i], __uint_as_float(s[q][i + 24]));
            }
          }
          mx = fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
        }
        float mul = 1.f;  // of a score, in the exponent
        if constexpr (MOD == 0) {
          mul = p.scale_log2;
          mx *= mul;  // -inf stays -inf
          // The exponent's multiply-add does not round its product, the maximum does: a
          // difference of powers of 2 once scores pass 2^24, of their sixteenths here.
          // Such rows' scores are rounded first, so that none passes the maximum.
          if (fabsf(mx) > 1048576.f && mx != kNegInf) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                s[c][e] = __float_as_uint(__fmul_rn(__uint_as_float(s[c][e]), mul));
            mul = 1.f;
          }
          __syncwarp();
        }
        // P of the last tile has been read, and O holds its product.
        ok = p_taken() && zero_pads(j, k0);
        if (!ok) break;
        ++sc;
        tc_fence_after();
        // Lazy maximum: the reference moves only when it falls 2^kLag behind a row's
        // maximum, which probabilities may reach until then. For FP16 it is set 2^7 below
        // the maximum: otherwise those below 2^-25 of the largest were rounded to 0, and
        // of tens of thousands of keys such ones can make a thousandth of the output.
        constexpr float kLift = std::is_same<T, __half>::value ? 7.f : 0.f, kLag = kLift + 8.f;
        float alpha = 1.f;
        bool rescale = false;
        if (mx - m_ref > kLag) {  // (no sum of them: past 2^24 that would round up)
          const float next = mx - kLift;
          alpha = fast_exp2(m_ref - next);
          rescale = m_ref != kNegInf;
          m_ref = next;
          l_sum *= alpha;
        }
        // O moves to the new reference (rare; eight columns at a time, the scores
        // being in registers).
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 8) {
            uint32_t o[8];
            tmem_ld8(tO + c, o);
            tmem_ld_wait();
            tmem_bind8(o);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st8(tO + c, o);
          }
          tmem_st_wait();
        }
        const float mb = m_ref == kNegInf ? 0.f : -m_ref;
        float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t ph[16];
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float x0, x1, x2, x3;
            fma_pair(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]),
                     mul, mb, x0, x1);
            fma_pair(__uint_as_float(s[c][e + 2]), __uint_as_float(s[c][e + 3]),
                     mul, mb, x2, x3);
            x0 = fast_exp2(x0);
            x1 = fast_exp2(x1);
            x2 = fast_exp2(x2);
            x3 = fast_exp2(x3);
            add_pair(l0, l1, x0, x1);
            add_pair(l2, l3, x2, x3);
            // (P in the input's 16 bits, as the A operand of a product with V has to be:
            // one rounding of half a step a term, no more than the output's own; the sum
            // l keeps the unrounded values)
            ph[e / 2] = pack_pair<T>(x0, x1);
            ph[e / 2 + 1] = pack_pair<T>(x2, x3);
            if constexpr (F32) {  // what the rounding took off (in the scores' place)
              const float2 h0 = unpack_pair<T>(ph[e / 2]), h1 = unpack_pair<T>(ph[e / 2 + 1]);
              s[c][e / 2] = pack_pair<T>(x0 - h0.x, x1 - h0.y);
              s[c][e / 2 + 1] = pack_pair<T>(x2 - h1.x, x3 - h1.y);
            }
          }
          tmem_st16(tP + c * 16, ph);
          if (c == 1) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_half[grp]);
          }
        }
        l_sum += (l0 + l1) + (l2 + l3);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[grp]);
        if constexpr (F32) {
          ++pn;
          ok = p_taken();
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pl[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) pl[e] = s[c][e];
            tmem_st16(tP + c * 16, pl);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&p_half[grp]);
            mbar_arrive(&p_full[grp]);
          }
          ++pn;
        }
      }
      if (!ok) break;
      tile0 += unsigned(d.nt);

      // -------------------------------------------------------------- epilogue
      ok = p_taken();
      if (!ok) break;
      tc_fence_after();
      // A row that saw keys, but no score above -inf: a reference of its own tells it
      // from one that saw none (its O is 0, its l 0, or NaN where a score was NaN).
      if (m_ref == kNegInf && max(lo, d.t0 * kChTile) < min(hi, min(d.hi, (d.t0 + d.nt) * kChTile)))
        m_ref = kLowest;
      // The row's factor on each group's O (0 where it saw no key), its columns
      // [c0, c1), and where they go.
      float f0, f1 = 0.f, m_out = m_ref, l_out = l_sum;
      int c0 = 0, c1 = D;
      if (!dual) {
        // (the other group's (m, l) come once its products are complete too)
        ml_x[grp * 128 + row] = make_float2(m_ref, l_sum);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&xch[grp]);
        ok = __all_sync(0xffffffffu, mbar_wait(&xch[grp ^ 1], alt & 1));
        if (!ok) break;
        tc_fence_after();
        const float2 a = ml_x[row], b = ml_x[128 + row];
        m_out = fmaxf(a.x, b.x);
        f0 = a.x == kNegInf ? 0.f : fast_exp2(a.x - m_out);
        f1 = b.x == kNegInf ? 0.f : fast_exp2(b.x - m_out);
        l_out = f0 * a.y + f1 * b.y;
        c0 = grp * (D / 2);
        c1 = c0 + D / 2;
      } else {
        f0 = m_ref == kNegInf ? 0.f : 1.f;
      }
      if (d.slot < 0) {
        const float inv = m_out == kNegInf ? 0.f : 1.f / l_out;  // (l of 0 or NaN: NaN below)
        f0 *= inv;
        f1 *= inv;
      }
      const bool two = !dual && d.nt > 1;  // group 1 has products of its own
      const uint32_t tA = tbase + lane_addr + G::kTmemO + (dual ? uint32_t(grp) * 128 : 0u);
      if (!idle) {
        const int prow = (dual ? grp * 128 : 0) + row;
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
          uint32_t o[32], o2[32];
          tmem_ld32(tA + c, o);
          if (two) tmem_ld32(tA + 128 + c, o2);
          tmem_ld_wait();
          tmem_bind32(o);
          float v[32];
          if (two) {
            tmem_bind32(o2);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              v[e] = (f0 != 0.f ? f0 * __uint_as_float(o[e]) : 0.f) +
                     (f1 != 0.f ? f1 * __uint_as_float(o2[e]) : 0.f);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = f0 != 0.f ? f0 * __uint_as_float(o[e]) : 0.f;
          }
          if (valid && d.slot >= 0) {
            float4* to = p.part_o + (size_t(d.slot) * (D / 4) + c / 4) * p.part_rows + prow;
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              to[size_t(e / 4) * p.part_rows] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          } else if (valid) {
            const size_t at = (size_t(d.first + tok) * p.hq + head) * D + c;
            if constexpr (F32) {
              float4* to = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                to[e / 4] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            } else {
              // (a thread's row lies apart from its neighbours': whole 32-byte sectors)
              T* to = static_cast<T*>(p.out) + at;
#pragma unroll
              for (int e = 0; e < 32; e += 16)
                st_global_v8(to + e, pack_pair<T>(v[e], v[e + 1]), pack_pair<T>(v[e + 2], v[e + 3]),
                             pack_pair<T>(v[e + 4], v[e + 5]), pack_pair<T>(v[e + 6], v[e + 7]),
                             pack_pair<T>(v[e + 8], v[e + 9]), pack_pair<T>(v[e + 10], v[e + 11]),
                             pack_pair<T>(v[e + 12], v[e + 13]), pack_pair<T>(v[e + 14], v[e + 15]));
            }
          }
          __syncwarp();
        }
        if (d.slot >= 0 && valid && (dual || grp == 0))
          p.part_ml[size_t(d.slot) * p.part_rows + prow] = make_float2(m_out, l_out);
      }
      tc_fence_before();
      if (!dual) {  // both groups read both O: neither goes on before the other has
        __syncwarp();
        if (lane == 0) mbar_arrive(&xch_done[grp]);
        ok = __all_sync(0xffffffffu, mbar_wait(&xch_done[grp ^ 1], alt & 1));
        ++alt;
        tc_fence_after();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&desc_empty[ds]);
    }
    if (!ok && lane == 0) atomicOr(p.err, kErrTimeout);
    tc_fence_before();
    named_barrier_sync(1, kChThreads);
  }
}

// Joins the pieces of the item that starts (and does not end) in block
// blockIdx.x: its own, then those of the following blocks up to the one that
// ends it, 32 rows per block of blockIdx.y.
template <int D, typename T>
__global__ void __launch_bounds__(kChMergeThreads) chunk_merge_kernel(const ChunkParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  grid_dependency_wait();
  const int c = blockIdx.x, blocks = gridDim.x;
  const int* s = p.sched + size_t(c) * 8;
  if (!s[1]) return;
  const int first = s[2], ntok = s[3], head = s[4];
  const int row = blockIdx.y * 32 + lane;
  const int tok = (row / 128) * p.tile_tokens + (row % 128) / p.group;
  const bool valid = row < p.part_rows && (row % 128) / p.group < p.tile_tokens && tok < ntok;
  if (!__any_sync(0xffffffffu, valid)) return;
  // Where the pieces lie, 32 blocks looked at together: those after c that have a
  // share, up to the one that ends the item.
  constexpr int kMost = 160;  // (a block per SM)
  __shared__ int s_slot[kChMergeThreads / 32][kMost];
  int* slot = s_slot[warp];
  int n = 1;
  if (lane == 0) slot[0] = c * 2 + 1;
  for (int i0 = c + 1;; i0 += 32) {
    const int state = i0 + lane < blocks ? p.sched[size_t(i0 + lane) * 8] : 2;
    const unsigned ends = __ballot_sync(0xffffffffu, state == 2);
    const unsigned upto = ends ? ends ^ (ends - 1) : 0xffffffffu;  // through the first end
    const unsigned has = __ballot_sync(0xffffffffu, state != 3 && i0 + lane < blocks) & upto;
    const int at = n + __popc(has & ((1u << lane) - 1));
    if ((has >> lane & 1) && at < kMost) slot[at] = (i0 + lane) * 2;
    n = min(n + __popc(has), kMost);
    if (ends) break;
  }
  __syncwarp();
  if (!valid) return;
  // Online over the pieces, in order, four pieces' loads in flight together.
  constexpr int N = D / 32;  // float4 pieces of a warp
  constexpr int F = 4;
  float m = -INFINITY, l = 0.f;
  float4 acc[N];
#pragma unroll
  for (int q = 0; q < N; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += F) {
    float2 ml[F];
    float4 o[F][N];
#pragma unroll
    for (int i = 0; i < F; ++i) {
      const bool in = i0 + i < n;
      const size_t at = in ? size_t(slot[i0 + i]) : 0;
      ml[i] = in ? p.part_ml[at * p.part_rows + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int q = 0; q < N; ++q)
        o[i][q] = in ? p.part_o[(at * (D / 4) + warp * N + q) * p.part_rows + row]
                     : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mn = m;
#pragma unroll
    for (int i = 0; i < F; ++i) mn = fmaxf(mn, ml[i].x);
    const float a = m == -INFINITY ? 0.f : fast_exp2(m - mn);
    m = mn;
    l *= a;
#pragma unroll
    for (int q = 0; q < N; ++q) {
      acc[q].x *= a;
      acc[q].y *= a;
      acc[q].z *= a;
      acc[q].w *= a;
    }
#pragma unroll
    for (int i = 0; i < F; ++i) {
      // (a piece without keys has O = 0)
      const float w = ml[i].x == -INFINITY ? 0.f : fast_exp2(ml[i].x - m);
      l += w * ml[i].y;
#pragma unroll
      for (int q = 0; q < N; ++q) {
        acc[q].x += w * o[i][q].x;
        acc[q].y += w * o[i][q].y;
        acc[q].z += w * o[i][q].z;
        acc[q].w += w * o[i][q].w;
      }
    }
  }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;
  const size_t at = (size_t(first + tok) * p.hq + head * p.group + (row % 128) % p.group) * D +
                    warp * N * 4;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const float4 o = make_float4(acc[q].x * inv, acc[q].y * inv, acc[q].z * inv, acc[q].w * inv);
    if (p.out_f32)
      *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at + q * 4) = o;
    else
      *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + at + q * 4) =
          make_uint2(pack_pair<T>(o.x, o.y), pack_pair<T>(o.z, o.w));
  }
}

}  // namespace bc
