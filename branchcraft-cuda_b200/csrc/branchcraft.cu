// Host side of libbranchcraft.so: argument validation (the reference's rules,
// src/paged_gqa.cu:122-132, src/tree_attention.cu:93-122,
// src/packed_decode.cu:64-82), TMA tensor-map encoding, launch-shape choice and
// the extern "C" entry points declared in include/branchcraft.h.
//
// The library is stateless with respect to its callers: it allocates nothing,
// launches only on the stream it is given and keeps just per-device caches of
// immutable facts (SM count, the error-word address, which kernels had their
// shared-memory limit raised).
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <mutex>
#include <utility>

#include "bc_append.cuh"
#include "bc_attn.cuh"
#include "bc_beam.cuh"
#include "bc_chunk.cuh"
#include "bc_commit.cuh"
#include "bc_cow_plan.cuh"
#include "bc_exchange.cuh"
#include "bc_tree_mma.cuh"
#include "branchcraft.h"

static_assert(bc::kCowPlanMaxNodes == BC_MAX_NODES, "the planner's node cap is the API's");
static_assert(bc::kAppendMaxBatch == BC_MAX_SEQUENCES && bc::kBeamMax == BC_MAX_BEAMS &&
                  bc::kBeamMaxVocab == BC_MAX_BEAM_VOCAB && bc::kChMaxBatch == BC_MAX_CHUNK_REQUESTS,
              "the kernels' limits are the API's");

namespace bc {

// Per-device error word (BC_ERR_* bits), set by kernels with atomicOr.
__device__ unsigned g_error_word;

namespace {

constexpr int kMaxDevices = 64;
constexpr float kLog2e = 1.4426950408889634f;

int current_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -1;
  return dev;
}

unsigned* error_word(int dev) {
  static std::atomic<unsigned*> cache[kMaxDevices];
  static std::mutex mu;
  unsigned* p = cache[dev].load(std::memory_order_acquire);
  if (p) return p;
  std::lock_guard<std::mutex> lock(mu);
  p = cache[dev].load(std::memory_order_relaxed);
  if (!p) {
    if (cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_error_word) != cudaSuccess)
      return nullptr;
    cache[dev].store(p, std::memory_order_release);
  }
  return p;
}

// A fresh abort token for each launch (never 0: 0 disables the abort check).
unsigned next_launch_token() {
  static std::atomic<unsigned> counter{0};
  unsigned t = counter.fetch_add(1, std::memory_order_relaxed) + 1;
  if (t == 0) t = counter.fetch_add(1, std::memory_order_relaxed) + 1;
  return t;
}

int sm_count(int dev) {
  static std::atomic<int> cache[kMaxDevices];
  int n = cache[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1)
    n = 148;
  cache[dev].store(n, std::memory_order_relaxed);
  return n;
}

// ------------------------------------------------------------ tensor maps
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                         &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return static_cast<EncodeTiledFn>(nullptr);
    return reinterpret_cast<EncodeTiledFn>(f);
  }();
  return fn;
}

// FP16 4-D map with a 64-element inner box and 128-byte swizzle.
bool encode_map(CUtensorMap* map, const void* base, const uint64_t dims[4],
                const uint64_t strides_bytes[3], const uint32_t box[4]) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  if (reinterpret_cast<uintptr_t>(base) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (strides_bytes[i] % 16 || strides_bytes[i] >= (uint64_t(1) << 40)) return false;
  cuuint64_t gdim[4] = {dims[0], dims[1], dims[2], dims[3]};
  cuuint64_t gstr[3] = {strides_bytes[0], strides_bytes[1], strides_bytes[2]};
  cuuint32_t bdim[4] = {box[0], box[1], box[2], box[3]};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), gdim, gstr, bdim,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// K or V of a paged cache viewed as 4-D (D, heads, 16 slots, pages) — or
// (D, 16 slots, heads, pages) when the slot stride is the smaller one — with
// strides given in elements.
bool encode_cache_map(CUtensorMap* map, const void* base, int dim, int heads, int pages,
                      long long head_stride, long long slot_stride, long long block_stride,
                      bool* slot_major) {
  *slot_major = slot_stride < head_stride;
  const uint64_t dims[4] = {uint64_t(dim), uint64_t(*slot_major ? 16 : heads),
                            uint64_t(*slot_major ? heads : 16), uint64_t(pages)};
  const uint64_t st[3] = {uint64_t(*slot_major ? slot_stride : head_stride) * 2,
                          uint64_t(*slot_major ? head_stride : slot_stride) * 2,
                          uint64_t(block_stride) * 2};
  const uint32_t box[4] = {64, uint32_t(*slot_major ? 16 : 1), uint32_t(*slot_major ? 1 : 16), 1};
  return encode_map(map, base, dims, st, box);
}

// Draft K or V [batch, nodes, heads, D] as 4-D (D, heads, nodes, batch).
bool encode_draft_map(CUtensorMap* map, const void* base, int dim, int heads, int nodes,
                      int batch) {
  const uint64_t dims[4] = {uint64_t(dim), uint64_t(heads), uint64_t(nodes), uint64_t(batch)};
  const uint64_t st[3] = {uint64_t(dim) * 2, uint64_t(heads) * dim * 2,
                          uint64_t(nodes) * heads * dim * 2};
  const uint32_t box[4] = {64, 1, 16, 1};
  return encode_map(map, base, dims, st, box);
}

// ---------------------------------------------------------------- launches
// FP32 merge of split partials, a programmatic dependent of the kernel that
// wrote them.
cudaError_t launch_merge(int dim, int rows, int splits, const float* pml, const float* pa,
                         float* out, cudaStream_t stream, int per_block = 0,
                         long long block_stride = 0, float* out_ml = nullptr) {
  if (per_block <= 0) per_block = splits;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((rows + 3) / 4), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (out_ml)  // merged state, not the normalised rows
    return dim == 64 ? cudaLaunchKernelEx(&cfg, merge_kernel<64, true>, rows, splits, per_block,
                                          block_stride, pml, pa, out, out_ml)
                     : cudaLaunchKernelEx(&cfg, merge_kernel<128, true>, rows, splits, per_block,
                                          block_stride, pml, pa, out, out_ml);
  return dim == 64 ? cudaLaunchKernelEx(&cfg, merge_kernel<64>, rows, splits, per_block,
                                        block_stride, pml, pa, out, out_ml)
                   : cudaLaunchKernelEx(&cfg, merge_kernel<128>, rows, splits, per_block,
                                        block_stride, pml, pa, out, out_ml);
}

template <int D, int RT, bool OUT_HALF>
cudaError_t launch_attn_t(const AttnParams& p, const CUtensorMap* maps, int items, int cluster,
                          cudaStream_t stream) {
  auto kern = attn_kernel<D, RT, OUT_HALF>;
  const size_t smem = AttnGeom<D>::kSmemBytes;
  static std::atomic<uint64_t> configured{0};
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (!(configured.load(std::memory_order_relaxed) & (uint64_t(1) << dev))) {
    cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    configured.fetch_or(uint64_t(1) << dev);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(items), 1, unsigned(p.splits));
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  // Programmatic dependent launch: scheduled while the preceding kernel
  // finishes, waiting for it before the first input read.
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = unsigned(cluster);
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kern, p, maps[0], maps[1]);
}

template <int D, bool OUT_HALF>
cudaError_t launch_attn_rt(int rt, const AttnParams& p, const CUtensorMap* maps, int items,
                           int cluster, cudaStream_t stream) {
  switch (rt) {
    case 1: return launch_attn_t<D, 1, OUT_HALF>(p, maps, items, cluster, stream);
    case 2: return launch_attn_t<D, 2, OUT_HALF>(p, maps, items, cluster, stream);
    default: return launch_attn_t<D, 4, OUT_HALF>(p, maps, items, cluster, stream);
  }
}

cudaError_t launch_attn(int dim, int rt, bool out_half, const AttnParams& p,
                        const CUtensorMap* maps, int items, int cluster, cudaStream_t stream) {
  if (dim == 64)
    return out_half ? launch_attn_rt<64, true>(rt, p, maps, items, cluster, stream)
                    : launch_attn_rt<64, false>(rt, p, maps, items, cluster, stream);
  return out_half ? launch_attn_rt<128, true>(rt, p, maps, items, cluster, stream)
                  : launch_attn_rt<128, false>(rt, p, maps, items, cluster, stream);
}

// Row tiling: RT 8-row tiles per CTA (1, 2 or 4) and the CTAs along the rows.
void row_tiling(int rows, int* rt, int* row_chunks) {
  *rt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  *row_chunks = (rows + 8 * *rt - 1) / (8 * *rt);
}

// Cluster split for one launch: split only to fill the GPU (two CTAs per SM),
// keep at least 8 pages per CTA, and never exceed 8 CTAs (the portable cluster
// size). Splitting large ragged batches for balance loses: a cluster needs all
// of its CTAs free at once inside one GPC, which leaves SMs idle.
int auto_cluster(long long items, int max_virtual_pages, int sms) {
  int c = 1;
  while (c < 8 && items * c < 2LL * sms) c *= 2;
  while (c > 1 && (max_virtual_pages + c - 1) / c < 8) c /= 2;
  return c;
}

bool basic_shape_ok(const bc_shape* s) {
  return s && s->batch >= 1 && s->query_heads >= 1 && s->kv_heads >= 1 &&
         s->query_heads % s->kv_heads == 0 && (s->dim == 64 || s->dim == 128) &&
         s->max_pages >= 1 && s->physical_pages >= 1;
}

AttnParams base_params(const bc_shape* s, unsigned* err) {
  AttnParams p = {};
  p.batch = s->batch;
  p.hq = s->query_heads;
  p.hkv = s->kv_heads;
  p.group = s->query_heads / s->kv_heads;
  p.max_pages = s->max_pages;
  p.physical_pages = s->physical_pages;
  p.rows = p.group;
  p.err = err;
  p.token = next_launch_token();
  return p;
}

// Paged decode core shared by bc_decode / bc_paged_decode / partial variants.
// mode: kSplitNone / kSplitCluster / kSplitGlobal; emit_partial stores one
// (m, l, acc) partial per (request, q-head).
cudaError_t paged_decode_core(const bc_shape* s, const void* q, const void* k, const void* v,
                              const int* pages, const int* lengths, void* out, bool out_half,
                              float scale, int splits, int mode, bool emit_partial,
                              float* partial_a, float* partial_ml, bool slot_major_hint,
                              const CUtensorMap* kv_maps, cudaStream_t stream) {
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  AttnParams p = base_params(s, err);
  int rt = 1;
  row_tiling(p.rows, &rt, &p.row_chunks);
  p.splits = splits;
  p.split_mode = mode;
  p.emit_partial = emit_partial ? 1 : 0;
  p.slot_major = slot_major_hint ? 1 : 0;
  p.q = static_cast<const __half*>(q);
  p.pages = pages;
  p.lengths = lengths;
  p.out = out;
  p.partial_a = partial_a;
  p.partial_ml = partial_ml;
  p.scale_log2 = scale * kLog2e;
  CUtensorMap maps[2];
  if (kv_maps) {
    maps[0] = kv_maps[0];
    maps[1] = kv_maps[1];
  } else {
    bool sm = false;
    const long long hs = s->dim, ss = (long long)s->kv_heads * s->dim, bs = 16 * ss;
    if (!encode_cache_map(&maps[0], k, s->dim, s->kv_heads, s->physical_pages, hs, ss, bs, &sm) ||
        !encode_cache_map(&maps[1], v, s->dim, s->kv_heads, s->physical_pages, hs, ss, bs, &sm))
      return cudaErrorInvalidValue;
    p.slot_major = sm ? 1 : 0;
  }
  const long long items = (long long)s->kv_heads * s->batch * p.row_chunks;
  if (items > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int cluster = mode == kSplitCluster ? splits : 1;
  cudaError_t e = launch_attn(s->dim, rt, out_half, p, maps, int(items), cluster, stream);
  if (e != cudaSuccess || mode != kSplitGlobal || emit_partial) return e;
  const int rows = s->batch * s->query_heads;
  return launch_merge(s->dim, rows, splits, partial_ml, partial_a, static_cast<float*>(out),
                      stream);
}

int pick_mode(int splits) { return splits <= 1 ? kSplitNone : splits <= 8 ? kSplitCluster : kSplitGlobal; }

template <int D, bool PREC, bool OUT_HALF, bool DUAL = false>
cudaError_t configure_tree_kernel(int dev) {
  static std::atomic<uint64_t> configured{0};
  if (configured.load(std::memory_order_relaxed) & (uint64_t(1) << dev)) return cudaSuccess;
  // The kernel's register split (setmaxnreg) hands out exactly the launch
  // budget of kTreeLaunchRegs per thread; with fewer registers at launch its
  // increase could never be granted, so such a build is refused here.
  cudaFuncAttributes fa;
  cudaError_t e = cudaFuncGetAttributes(&fa, tree_mma_kernel<D, PREC, OUT_HALF, DUAL>);
  if (e != cudaSuccess) return e;
  if (fa.numRegs != kTreeLaunchRegs) return cudaErrorInvalidDeviceFunction;
  const size_t most = TreeGeom<D, PREC, DUAL>::smem_bytes(BC_MAX_NODES);
  e = cudaFuncSetAttribute(tree_mma_kernel<D, PREC, OUT_HALF, DUAL>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, int(most));
  if (e != cudaSuccess) return e;
  configured.fetch_or(uint64_t(1) << dev);
  return cudaSuccess;
}

// How many clusters of `c` CTAs of this kernel can be resident at once (one
// CTA per SM at this shared-memory size); cached per device and size.
template <int D, bool PREC, bool OUT_HALF>
int tree_max_clusters(int dev, int c) {
  static std::atomic<int> cache[kMaxDevices][9];
  const int slot = c;  // 1..8
  int n = cache[dev][slot].load(std::memory_order_relaxed);
  if (n > 0) return n;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, unsigned(c));
  cfg.blockDim = dim3(kTreeThreads, 1, 1);
  cfg.dynamicSmemBytes = TreeGeom<D, PREC>::smem_bytes(BC_MAX_NODES);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = unsigned(c);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (configure_tree_kernel<D, PREC, OUT_HALF>(dev) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, tree_mma_kernel<D, PREC, OUT_HALF>, &cfg) !=
          cudaSuccess ||
      n < 1) {
    cudaGetLastError();
    n = sm_count(dev) / c;
  }
  cache[dev][slot].store(n, std::memory_order_relaxed);
  return n;
}

// Cluster split along the keys: the largest size (any of 1..8) whose CTAs fit
// on the SMs in one wave of resident clusters, with at least two key tiles per
// CTA. A small batch needs every SM it can get: each CTA's copy rate, not the
// memory, bounds it.
template <int D, bool PREC, bool OUT_HALF>
int tree_splits(int dev, long long items, int tiles) {
  const int sms = sm_count(dev);
  int c = int(std::min<long long>(8, std::max<long long>(1, sms / std::max<long long>(items, 1))));
  while (c > 1 && (items > tree_max_clusters<D, PREC, OUT_HALF>(dev, c) || (tiles + c - 1) / c < 2))
    --c;
  return c;
}

// The planner as its own single-CTA launch (a programmatic dependent).
cudaError_t launch_cow_plan(const CowPlanParams& p, cudaStream_t stream) {
  const size_t smem = cow_plan_smem_bytes(p.batch);
  static std::atomic<uint64_t> configured{0};
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (!(configured.load(std::memory_order_relaxed) & (uint64_t(1) << dev))) {
    const cudaError_t e = cudaFuncSetAttribute(
        cow_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
        int(cow_plan_smem_bytes(kCowPlanMaxBatch)));
    if (e != cudaSuccess) return e;
    configured.fetch_or(uint64_t(1) << dev);
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, 1, 1);
  cfg.blockDim = dim3(kCowPlanThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, cow_plan_kernel, p);
}

template <int D, bool PREC, bool OUT_HALF, bool DUAL>
cudaError_t launch_tree_t(TreeParams& p, const CUtensorMap* maps, int items, int tiles,
                          size_t smem, cudaStream_t stream) {
  auto kern = tree_mma_kernel<D, PREC, OUT_HALF, DUAL>;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  cudaError_t e = configure_tree_kernel<D, PREC, OUT_HALF, DUAL>(dev);
  if (e != cudaSuccess) return e;
  // A DUAL grid has several waves by construction: never split.
  p.splits = DUAL ? 1 : tree_splits<D, PREC, OUT_HALF>(dev, items, tiles);
  // One CTA per SM: a cluster split fits one wave by construction, an
  // unsplit grid when it has no more CTAs than SMs.
  p.early_trigger = (p.splits > 1 || items <= sm_count(dev)) ? 1 : 0;
  int grid_items = items;
  if (p.plan_inline == 2) {
    // A device plan was asked for: made by one extra cluster of this launch
    // when the grid, that cluster included, is one wave (every CTA resident:
    // the verification CTAs can wait for the planner), else by the planner
    // launch, which this one then follows as a programmatic dependent.
    const bool wave = !DUAL && (p.splits > 1
                                    ? items + 1 <= tree_max_clusters<D, PREC, OUT_HALF>(dev, p.splits)
                                    : items + 1 <= sm_count(dev));
    if (wave && cow_plan_smem_bytes(p.plan.batch) + 1024 <= smem) {
      p.plan_inline = 1;
      p.plan_item = items;
      grid_items = items + 1;
    } else {
      p.plan_inline = 0;
      const cudaError_t e2 = launch_cow_plan(p.plan, stream);
      if (e2 != cudaSuccess) return e2;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid_items), 1, unsigned(p.splits));
  cfg.blockDim = dim3(kTreeThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  // Programmatic dependent launch: the CTAs may be scheduled while the
  // preceding kernel finishes; they wait for it before their first load.
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (p.splits > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = unsigned(p.splits);
    cfg.numAttrs = 2;
  }
  return cudaLaunchKernelEx(&cfg, kern, p, maps[0], maps[1], maps[2], maps[3]);
}

// Tree verification on tcgen05. Requests are grouped R to a 128-row tile
// (R = 128 / (nodes * group)); a group whose page tables match shares each
// K/V tile of the prefix. FP32 output accumulates P as FP16 hi + lo (FP32-exact
// products); FP16 output uses one FP16 P, matching its own rounding.
// The batch commit fused into a tree launch (bc_tree_verify_commit).
struct FusedCommit {
  const int *clone_src, *clone_dst, *entry_request, *entry_node, *entry_page, *entry_slot;
  int nclones, nentries;         // counts, or the capacities of a device-made plan
  const int* plan_counts;        // device-made plan: [clones, entries, status]
  const CowPlanParams* plan;     // the plan to make first (bc_tree_step)
};

cudaError_t tree_core(const bc_shape* s, const void* draft_q, const void* prefix_k,
                      const void* prefix_v, const int* pages, const int* lengths,
                      const void* draft_k, const void* draft_v, const int* parent, void* out,
                      bool out_half, int nodes, cudaStream_t stream,
                      const FusedCommit* commit = nullptr) {
  if (!basic_shape_ok(s) || nodes < 1 || nodes > BC_MAX_NODES || !prefix_k || !prefix_v ||
      !pages || !lengths || !draft_q || !draft_k || !draft_v || !parent || !out)
    return cudaErrorInvalidValue;
  if (commit) {
    const FusedCommit& c = *commit;
    if (c.nclones < 0 || c.nclones > 256 || c.nentries < 0 ||
        (c.nclones > 0 && (!c.clone_src || !c.clone_dst)) ||
        (c.nentries > 0 && (!c.entry_request || !c.entry_node || !c.entry_page || !c.entry_slot)) ||
        ((reinterpret_cast<uintptr_t>(prefix_k) | reinterpret_cast<uintptr_t>(prefix_v) |
          reinterpret_cast<uintptr_t>(draft_k) | reinterpret_cast<uintptr_t>(draft_v)) % 16))
      return cudaErrorInvalidValue;
  }
  if ((reinterpret_cast<uintptr_t>(draft_q) | reinterpret_cast<uintptr_t>(out)) % 16)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  TreeParams p = {};
  p.batch = s->batch;
  p.hq = s->query_heads;
  p.hkv = s->kv_heads;
  p.group = s->query_heads / s->kv_heads;
  p.nodes = nodes;
  p.max_pages = s->max_pages;
  p.physical_pages = s->physical_pages;
  p.rows_req = nodes * p.group;
  int R = p.rows_req >= kTreeRows ? 1 : kTreeRows / p.rows_req;
  R = std::min(R, std::min(s->batch, kTreeMaxReq));
  p.req_per_block = R;
  p.tiles_per_block = (R * p.rows_req + kTreeRows - 1) / kTreeRows;
  p.blocks = (s->batch + R - 1) / R;
  long long items = (long long)s->kv_heads * p.blocks * p.tiles_per_block;
  // Blocks of an even number of row tiles, in a grid of at least two waves
  // even after pairing: one CTA runs two row tiles over each K/V tile (half
  // the copies per FLOP). Small grids keep one row tile per CTA and split
  // the keys instead.
  const bool dual = p.tiles_per_block % 2 == 0 && items / 2 >= 2LL * sm_count(dev);
  if (dual) {
    p.tiles_per_block /= 2;
    items /= 2;
  }
  if (items > 0x7fffffffLL) return cudaErrorInvalidValue;
  // Key tiles of one CTA before splitting: prefix tiles plus draft tiles.
  const int npad = (nodes + 15) & ~15;
  const int tiles = (s->max_pages * kPageSize + kTreeTile - 1) / kTreeTile +
                    (R * npad + kTreeTile - 1) / kTreeTile;
  p.q = static_cast<const __half*>(draft_q);
  p.pages = pages;
  p.lengths = lengths;
  p.parent = parent;
  p.out = out;
  p.scale_log2 = kLog2e / std::sqrt(float(s->dim));
  p.err = err;
  p.token = next_launch_token();
  if (commit) {
    p.nclones = commit->nclones;
    p.nentries = commit->nentries;
    p.commit_tasks = 8 * commit->nclones + commit->nentries;
    p.plan_counts = commit->plan_counts;
    if (commit->plan) {
      p.plan = *commit->plan;
      p.plan_inline = 2;  // (launch_tree_t decides: inside this launch or before it)
    }
    p.cache_k = static_cast<__half*>(const_cast<void*>(prefix_k));
    p.cache_v = static_cast<__half*>(const_cast<void*>(prefix_v));
    p.draft_k = static_cast<const __half*>(draft_k);
    p.draft_v = static_cast<const __half*>(draft_v);
    p.clone_src = commit->clone_src;
    p.clone_dst = commit->clone_dst;
    p.entry_request = commit->entry_request;
    p.entry_node = commit->entry_node;
    p.entry_page = commit->entry_page;
    p.entry_slot = commit->entry_slot;
  }
  CUtensorMap maps[4];
  bool sm = false;
  const long long hs = s->dim, ss = (long long)s->kv_heads * s->dim, bs = 16 * ss;
  if (!encode_cache_map(&maps[0], prefix_k, s->dim, s->kv_heads, s->physical_pages, hs, ss, bs,
                        &sm) ||
      !encode_cache_map(&maps[1], prefix_v, s->dim, s->kv_heads, s->physical_pages, hs, ss, bs,
                        &sm) ||
      !encode_draft_map(&maps[2], draft_k, s->dim, s->kv_heads, nodes, s->batch) ||
      !encode_draft_map(&maps[3], draft_v, s->dim, s->kv_heads, nodes, s->batch))
    return cudaErrorInvalidValue;
  const int anc_rows = R * nodes;
  const int it = int(items);
  if (s->dim == 64) {
    if (dual)
      return out_half ? launch_tree_t<64, false, true, true>(p, maps, it, tiles, TreeGeom<64, false, true>::smem_bytes(anc_rows), stream)
                      : launch_tree_t<64, true, false, true>(p, maps, it, tiles, TreeGeom<64, true, true>::smem_bytes(anc_rows), stream);
    return out_half ? launch_tree_t<64, false, true, false>(p, maps, it, tiles, TreeGeom<64, false>::smem_bytes(anc_rows), stream)
                    : launch_tree_t<64, true, false, false>(p, maps, it, tiles, TreeGeom<64, true>::smem_bytes(anc_rows), stream);
  }
  if (dual)
    return out_half ? launch_tree_t<128, false, true, true>(p, maps, it, tiles, TreeGeom<128, false, true>::smem_bytes(anc_rows), stream)
                    : launch_tree_t<128, true, false, true>(p, maps, it, tiles, TreeGeom<128, true, true>::smem_bytes(anc_rows), stream);
  return out_half ? launch_tree_t<128, false, true, false>(p, maps, it, tiles, TreeGeom<128, false>::smem_bytes(anc_rows), stream)
                  : launch_tree_t<128, true, false, false>(p, maps, it, tiles, TreeGeom<128, true>::smem_bytes(anc_rows), stream);
}

// Self-test of the bounded waits: every CTA waits on an mbarrier that no
// one arrives at, with a short limit. The first wait to give up records the
// launch's abort token; the CTAs of later waves then give up at their first
// check. `smem` bytes of dynamic shared memory per CTA control how many CTAs
// share an SM (hence the waves).
__global__ void __launch_bounds__(32) selftest_wait_kernel(unsigned long long limit_ns,
                                                           unsigned token, unsigned* err) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    s_launch_token = token;
    mbar_init(&bar, 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (!__all_sync(0xffffffffu, mbar_wait(&bar, 0, limit_ns)) && threadIdx.x == 0)
    atomicOr(err, kErrTimeout);
}

}  // namespace
}  // namespace bc

using namespace bc;

extern "C" {

int bc_decode(const bc_shape* s, const void* q, const void* k, const void* v, const int* pages,
              const int* lengths, float* output, float* partial_a, float* partial_ml, int splits,
              void* stream) {
  if (!basic_shape_ok(s) || splits < 1 || splits > BC_MAX_SPLITS || !q || !k || !v || !pages ||
      !lengths || !output || (splits > 1 && (!partial_a || !partial_ml)))
    return cudaErrorInvalidValue;
  return paged_decode_core(s, q, k, v, pages, lengths, output, false,
                           1.0f / std::sqrt(float(s->dim)), splits, pick_mode(splits), false,
                           partial_a, partial_ml, false, nullptr,
                           static_cast<cudaStream_t>(stream));
}

int bc_auto_splits(const bc_shape* s, int max_length, int sm_count_arg) {
  if (!s || max_length < 512) return 1;
  const int groups = s->kv_heads > 0 ? s->kv_heads : 1;
  const int g = s->kv_heads > 0 ? s->query_heads / s->kv_heads : 1;
  int rt = 1, chunks = 1;
  row_tiling(g < 1 ? 1 : g, &rt, &chunks);
  const long long base = (long long)(s->batch > 0 ? s->batch : 1) * groups * chunks;
  // As many splits as make one wave of CTAs (two resident per SM): a second,
  // partial wave costs more than the longer key range of fewer splits. Any
  // count works (the merge takes 1..64); each split keeps >= 256 keys.
  const long long wave = 2LL * (sm_count_arg > 0 ? sm_count_arg : 148);
  long long splits = std::max(1LL, std::min<long long>(BC_MAX_SPLITS, wave / base));
  splits = std::min<long long>(splits, std::max(1, max_length / 256));
  return int(splits);
}

int bc_paged_decode(const bc_shape* s, const void* q, const void* k, const void* v,
                    const int* pages, const int* lengths, float* output, int splits,
                    void* stream) {
  if (!basic_shape_ok(s) || splits > 8 || !q || !k || !v || !pages || !lengths || !output)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (splits <= 0) {
    int rt = 1, chunks = 1;
    row_tiling(s->query_heads / s->kv_heads, &rt, &chunks);
    splits = auto_cluster((long long)s->batch * s->kv_heads * chunks, s->max_pages, sm_count(dev));
  }
  return paged_decode_core(s, q, k, v, pages, lengths, output, false,
                           1.0f / std::sqrt(float(s->dim)), splits, pick_mode(splits), false,
                           nullptr, nullptr, false, nullptr, static_cast<cudaStream_t>(stream));
}

int bc_paged_decode_partial(const bc_shape* s, const void* q, const void* k, const void* v,
                            const int* pages, const int* lengths, float* partial_ml,
                            float* partial_a, int splits, void* stream) {
  if (!basic_shape_ok(s) || splits > BC_MAX_SPLITS || !q || !k || !v || !pages || !lengths ||
      !partial_ml || !partial_a)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (splits <= 0) {
    int rt = 1, chunks = 1;
    row_tiling(s->query_heads / s->kv_heads, &rt, &chunks);
    splits = auto_cluster((long long)s->batch * s->kv_heads * chunks, s->max_pages, sm_count(dev));
  }
  // 1..8: merged inside a cluster, one partial per row. Above 8: every split
  // stores its own partial (global mode with the merge kernel left out).
  const int mode = splits <= 1 ? kSplitNone : splits <= 8 ? kSplitCluster : kSplitGlobal;
  return paged_decode_core(s, q, k, v, pages, lengths, nullptr, false,
                           1.0f / std::sqrt(float(s->dim)), splits, mode, true, partial_a,
                           partial_ml, false, nullptr, static_cast<cudaStream_t>(stream));
}

int bc_tree_verify(const bc_shape* s, const void* draft_q, const void* prefix_k,
                   const void* prefix_v, const int* pages, const int* lengths,
                   const void* draft_k, const void* draft_v, const int* parent, float* output,
                   int nodes, void* stream) {
  return tree_core(s, draft_q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent,
                   output, false, nodes, static_cast<cudaStream_t>(stream));
}

int bc_tree_verify_f16(const bc_shape* s, const void* draft_q, const void* prefix_k,
                       const void* prefix_v, const int* pages, const int* lengths,
                       const void* draft_k, const void* draft_v, const int* parent,
                       void* output_f16, int nodes, void* stream) {
  return tree_core(s, draft_q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent,
                   output_f16, true, nodes, static_cast<cudaStream_t>(stream));
}

int bc_tree_verify_commit(const bc_shape* s, const void* draft_q, void* cache_k, void* cache_v,
                          const int* pages, const int* lengths, const void* draft_k,
                          const void* draft_v, const int* parent, void* output, int output_f16,
                          int nodes, const int* clone_src, const int* clone_dst, int nclones,
                          const int* entry_request, const int* entry_node,
                          const int* entry_page, const int* entry_slot, int nentries,
                          void* stream) {
  const FusedCommit c{clone_src, clone_dst, entry_request, entry_node, entry_page, entry_slot,
                      nclones, nentries, nullptr, nullptr};
  return tree_core(s, draft_q, cache_k, cache_v, pages, lengths, draft_k, draft_v, parent,
                   output, output_f16 != 0, nodes, static_cast<cudaStream_t>(stream), &c);
}

int bc_cow_plan(int batch, int nodes, int physical_pages, const int* pages_in,
                int max_pages_in, const int* lengths_in, const int* path_len,
                const int* path_nodes, const int* refcount_in, const int* free_stack_in,
                const int* free_count_in, int* refcount, int* free_stack, int* free_count,
                int* pages_out, int max_pages_out, int* lengths_out, int* clone_src,
                int* clone_dst, int* entry_request, int* entry_node, int* entry_page,
                int* entry_slot, int* counts, void* stream) {
  if (batch < 1 || batch > kCowPlanMaxBatch || nodes < 1 || nodes > BC_MAX_NODES ||
      physical_pages < 1 || max_pages_in < 1 || max_pages_out < 1 ||
      !pages_in || !lengths_in || !path_len || !path_nodes || !refcount_in || !free_stack_in ||
      !free_count_in || !refcount || !free_stack || !free_count || !pages_out || !lengths_out || !clone_src || !clone_dst || !entry_request ||
      !entry_node || !entry_page || !entry_slot || !counts ||
      (long long)batch * nodes > 0x7fffffffLL || (long long)batch * max_pages_out > 0x7fffffffLL)
    return cudaErrorInvalidValue;
  const CowPlanParams p{batch, nodes, physical_pages, max_pages_in, max_pages_out, pages_in,
                        lengths_in, path_len, path_nodes, refcount_in, free_stack_in,
                        free_count_in, refcount, free_stack, free_count, pages_out,
                        lengths_out, clone_src, clone_dst, entry_request, entry_node,
                        entry_page, entry_slot, counts};
  return launch_cow_plan(p, static_cast<cudaStream_t>(stream));
}

int bc_tree_step(const bc_shape* s, const void* draft_q, void* cache_k, void* cache_v,
                 const int* pages, const int* lengths, const void* draft_k, const void* draft_v,
                 const int* parent, void* output, int output_f16, int nodes, const int* path_len,
                 const int* path_nodes, const int* refcount_in, const int* free_stack_in,
                 const int* free_count_in, int* refcount, int* free_stack, int* free_count,
                 int* pages_out, int max_pages_out, int* lengths_out, int* clone_src,
                 int* clone_dst, int* entry_request, int* entry_node, int* entry_page,
                 int* entry_slot, int* counts, void* stream) {
  if (!basic_shape_ok(s) || s->batch > kCowPlanMaxBatch || nodes < 1 || nodes > BC_MAX_NODES ||
      max_pages_out < 1 || !path_len || !path_nodes ||
      !refcount_in || !free_stack_in || !free_count_in || !refcount || !free_stack ||
      !free_count || !pages_out || !lengths_out || !clone_src || !clone_dst || !entry_request ||
      !entry_node || !entry_page || !entry_slot || !counts)
    return cudaErrorInvalidValue;
  const CowPlanParams plan{s->batch, nodes, s->physical_pages, s->max_pages, max_pages_out,
                           pages, lengths, path_len, path_nodes, refcount_in, free_stack_in,
                           free_count_in, refcount, free_stack, free_count, pages_out,
                           lengths_out, clone_src, clone_dst, entry_request, entry_node,
                           entry_page, entry_slot, counts};
  const FusedCommit c{clone_src, clone_dst, entry_request, entry_node, entry_page, entry_slot,
                      s->batch, s->batch * nodes, counts, &plan};
  return tree_core(s, draft_q, cache_k, cache_v, pages, lengths, draft_k, draft_v, parent,
                   output, output_f16 != 0, nodes, static_cast<cudaStream_t>(stream), &c);
}

int bc_packed_decode_kv(const bc_shape* s, const void* q, const void* packed_kv,
                        const int* pages, const int* lengths, void* output,
                        long long block_stride, long long head_stride, long long slot_stride,
                        long long kv_offset, float scale, int splits, void* stream) {
  if (!basic_shape_ok(s) || !q || !packed_kv || !pages || !lengths || !output ||
      block_stride < 1 || head_stride < 1 || slot_stride < 1 || !(scale > 0.f) || splits > 8)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  CUtensorMap maps[2];
  bool sm = false;
  const __half* kbase = static_cast<const __half*>(packed_kv);
  if (!encode_cache_map(&maps[0], kbase, s->dim, s->kv_heads, s->physical_pages, head_stride,
                        slot_stride, block_stride, &sm) ||
      !encode_cache_map(&maps[1], kbase + kv_offset, s->dim, s->kv_heads, s->physical_pages,
                        head_stride, slot_stride, block_stride, &sm))
    return cudaErrorInvalidValue;
  if (splits <= 0) {
    int rt = 1, chunks = 1;
    row_tiling(s->query_heads / s->kv_heads, &rt, &chunks);
    splits = auto_cluster((long long)s->batch * s->kv_heads * chunks, s->max_pages, sm_count(dev));
  }
  return paged_decode_core(s, q, nullptr, nullptr, pages, lengths, output, true, scale, splits,
                           splits > 1 ? kSplitCluster : kSplitNone, false, nullptr, nullptr, sm,
                           maps, static_cast<cudaStream_t>(stream));
}

int bc_packed_decode(const bc_shape* s, const void* q, const void* packed_kv, const int* pages,
                     const int* lengths, void* output, long long block_stride,
                     long long head_stride, long long slot_stride, float scale, void* stream) {
  if (!s) return cudaErrorInvalidValue;
  return bc_packed_decode_kv(s, q, packed_kv, pages, lengths, output, block_stride, head_stride,
                             slot_stride, s->dim, scale, 0, stream);
}

int bc_commit_path(const bc_shape* s, const void* draft_k, const void* draft_v, void* cache_k,
                   void* cache_v, const int* path_nodes, const int* dest_pages,
                   const int* dest_slots, int request, int nodes, int accepted, void* stream) {
  if (!s || !draft_k || !draft_v || !cache_k || !cache_v || !path_nodes || !dest_pages ||
      !dest_slots || request < 0 || request >= s->batch || nodes < 1 || accepted < 1 ||
      accepted > nodes || s->kv_heads < 1 || (s->dim != 64 && s->dim != 128))
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  const int row = s->kv_heads * s->dim;
  const bool vec = ((reinterpret_cast<uintptr_t>(draft_k) | reinterpret_cast<uintptr_t>(draft_v) |
                     reinterpret_cast<uintptr_t>(cache_k) | reinterpret_cast<uintptr_t>(cache_v)) %
                    16) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int physical = s->physical_pages > 0 ? s->physical_pages : 0x7fffffff;
  if (vec)
    commit_kernel<true><<<accepted, 256, 0, st>>>(
        row, s->batch, nodes, physical, static_cast<const __half*>(draft_k),
        static_cast<const __half*>(draft_v), static_cast<__half*>(cache_k),
        static_cast<__half*>(cache_v), nullptr, path_nodes, dest_pages, dest_slots, request, err);
  else
    commit_kernel<false><<<accepted, 256, 0, st>>>(
        row, s->batch, nodes, physical, static_cast<const __half*>(draft_k),
        static_cast<const __half*>(draft_v), static_cast<__half*>(cache_k),
        static_cast<__half*>(cache_v), nullptr, path_nodes, dest_pages, dest_slots, request, err);
  return cudaGetLastError();
}

int bc_commit_batch(const bc_shape* s, int nodes, const void* draft_k, const void* draft_v,
                    void* cache_k, void* cache_v, const int* clone_src, const int* clone_dst,
                    int nclones, const int* entry_request, const int* entry_node,
                    const int* entry_page, const int* entry_slot, int nentries, void* stream) {
  if (!s || !draft_k || !draft_v || !cache_k || !cache_v || nodes < 1 || nclones < 0 ||
      nentries < 0 || s->kv_heads < 1 || (s->dim != 64 && s->dim != 128) ||
      s->physical_pages < 1 || s->batch < 1 || (nclones > 0 && (!clone_src || !clone_dst)) ||
      (nentries > 0 && (!entry_request || !entry_node || !entry_page || !entry_slot)))
    return cudaErrorInvalidValue;
  const uintptr_t mis = (reinterpret_cast<uintptr_t>(draft_k) | reinterpret_cast<uintptr_t>(draft_v) |
                         reinterpret_cast<uintptr_t>(cache_k) | reinterpret_cast<uintptr_t>(cache_v)) %
                        16;
  if (mis) return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int row = s->kv_heads * s->dim;
  // Programmatic dependent launches: scheduled while the kernel before them
  // finishes, waiting for it before the first read.
  cudaLaunchAttribute pdl[1];
  pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = st;
  cfg.attrs = pdl;
  cfg.numAttrs = 1;
  if (nclones + nentries == 0) return cudaSuccess;
  if (nclones <= 256) {  // one launch (each entry CTA lists at most 256 clones)
    cfg.gridDim = dim3(unsigned(8 * nclones + nentries), 1, 1);
    return cudaLaunchKernelEx(&cfg, commit_batch_kernel, row, s->batch, nodes, s->physical_pages,
                              static_cast<const __half*>(draft_k),
                              static_cast<const __half*>(draft_v), static_cast<__half*>(cache_k),
                              static_cast<__half*>(cache_v), clone_src, clone_dst, nclones,
                              entry_request, entry_node, entry_page, entry_slot, nentries, err);
  }
  // Larger batches: every clone, then every row commit.
  if (nclones > 0) {
    cfg.gridDim = dim3(4, unsigned(nclones), 2);
    cudaError_t e = cudaLaunchKernelEx(&cfg, clone_kernel, 16 * row, s->physical_pages,
                                       static_cast<__half*>(cache_k),
                                       static_cast<__half*>(cache_v), clone_src, clone_dst, err);
    if (e != cudaSuccess) return e;
  }
  if (nentries > 0) {
    cfg.gridDim = dim3(unsigned(nentries), 1, 1);
    return cudaLaunchKernelEx(&cfg, commit_kernel<true>, row, s->batch, nodes,
                              s->physical_pages, static_cast<const __half*>(draft_k),
                              static_cast<const __half*>(draft_v), static_cast<__half*>(cache_k),
                              static_cast<__half*>(cache_v), entry_request, entry_node,
                              entry_page, entry_slot, 0, err);
  }
  return cudaSuccess;
}

int bc_merge_partials(int splits, int rows, int dim, const float* partial_ml,
                      const float* partial_a, float* out, void* stream) {
  if (splits < 1 || rows < 1 || (dim != 64 && dim != 128) || !partial_ml || !partial_a || !out)
    return cudaErrorInvalidValue;
  return launch_merge(dim, rows, splits, partial_ml, partial_a, out,
                      static_cast<cudaStream_t>(stream));
}

int bc_merge_to_partial(int splits, int rows, int dim, const float* partial_ml,
                        const float* partial_a, float* out_ml, float* out_a, void* stream) {
  if (splits < 1 || rows < 1 || (dim != 64 && dim != 128) || !partial_ml || !partial_a ||
      !out_ml || !out_a)
    return cudaErrorInvalidValue;
  return launch_merge(dim, rows, splits, partial_ml, partial_a, out_a,
                      static_cast<cudaStream_t>(stream), 0, 0, out_ml);
}

size_t bc_exchange_bytes(int world, int rows, int dim) {
  if (world < 1 || world > BC_MAX_EXCHANGE_RANKS || rows < 1 || (dim != 64 && dim != 128))
    return 0;
  return dim == 64 ? Exch<64>::bytes(world, rows) : Exch<128>::bytes(world, rows);
}

int bc_exchange_create(int world, int rows, int dim, void** buffer, void* ipc_handle) {
  const size_t n = bc_exchange_bytes(world, rows, dim);
  if (n == 0 || !buffer || !ipc_handle) return cudaErrorInvalidValue;
  void* p = nullptr;
  cudaError_t e = cudaMalloc(&p, n);
  if (e != cudaSuccess) return e;
  // zero flags: no epoch (>= 1) is published yet
  e = cudaMemset(p, 0, n);
  if (e == cudaSuccess) e = cudaIpcGetMemHandle(static_cast<cudaIpcMemHandle_t*>(ipc_handle), p);
  if (e != cudaSuccess) {
    cudaFree(p);
    return e;
  }
  *buffer = p;
  return cudaSuccess;
}

int bc_exchange_open(const void* ipc_handle, void** peer_buffer) {
  if (!ipc_handle || !peer_buffer) return cudaErrorInvalidValue;
  cudaIpcMemHandle_t h;
  std::memcpy(&h, ipc_handle, sizeof(h));
  return cudaIpcOpenMemHandle(peer_buffer, h, cudaIpcMemLazyEnablePeerAccess);
}

int bc_exchange_close(void* peer_buffer) {
  return peer_buffer ? cudaIpcCloseMemHandle(peer_buffer) : cudaErrorInvalidValue;
}

int bc_exchange_destroy(void* buffer) { return buffer ? cudaFree(buffer) : cudaErrorInvalidValue; }

int bc_merge_exchange(int world, int rank, unsigned epoch, int splits, int rows, int dim,
                      const float* partial_ml, const float* partial_a, float* const* peer_buffers,
                      float* out, void* stream) {
  if (world < 1 || world > BC_MAX_EXCHANGE_RANKS || rank < 0 || rank >= world || epoch == 0 ||
      splits < 1 || rows < 1 || (dim != 64 && dim != 128) || !partial_ml || !partial_a ||
      !peer_buffers || !out)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned((rows + kExchRowsPerBlock - 1) / kExchRowsPerBlock), 1, 1);
  cfg.blockDim = dim3(32 * kExchRowsPerBlock, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const unsigned token = next_launch_token();
  return dim == 64
             ? cudaLaunchKernelEx(&cfg, exchange_merge_kernel<64>, world, rank, epoch, splits, rows,
                                  partial_ml, partial_a, peer_buffers, out, token, err)
             : cudaLaunchKernelEx(&cfg, exchange_merge_kernel<128>, world, rank, epoch, splits,
                                  rows, partial_ml, partial_a, peer_buffers, out, token, err);
}

int bc_merge_gathered(int world, int splits, int rows, int dim, const float* gathered,
                      float* out, void* stream) {
  if (world < 1 || splits < 1 || rows < 1 || (dim != 64 && dim != 128) || !gathered || !out ||
      (long long)world * splits > 0x7fffffffLL)
    return cudaErrorInvalidValue;
  // rank r's block: splits*rows (m, l) pairs, then splits*rows*dim accumulators
  const long long ml_floats = (long long)splits * rows * 2;
  const long long block = ml_floats + (long long)splits * rows * dim;
  return launch_merge(dim, rows, world * splits, gathered, gathered + ml_floats, out,
                      static_cast<cudaStream_t>(stream), splits, block);
}

// ---------------------------------------------------------------------------
// Allocation-free decode: split partials in a library-owned device array.
// ---------------------------------------------------------------------------
}  // extern "C"

namespace {

// The array is a device symbol: host code must use its device address, which
// cudaGetSymbolAddress returns for the device that is current at the call.
static __device__ __align__(256) float bc_static_decode_scratch[BC_STATIC_SCRATCH_FLOATS];

// The array's device address on `dev` (current), looked up once per device.
// A failed look-up returns its own error code and clears it from the
// runtime's last-error slot, so the caller's next cudaGetLastError() does not
// report it a second time.
cudaError_t static_scratch_address(int dev, float** out) {
  static std::atomic<float*> cache[kMaxDevices];
  static std::mutex mu;
  float* p = cache[dev].load(std::memory_order_acquire);
  if (!p) {
    std::lock_guard<std::mutex> lock(mu);
    p = cache[dev].load(std::memory_order_relaxed);
    if (!p) {
      void* addr = nullptr;
      const cudaError_t e = cudaGetSymbolAddress(&addr, bc_static_decode_scratch);
      if (e != cudaSuccess || !addr) {
        cudaGetLastError();
        return e != cudaSuccess ? e : cudaErrorInvalidDevice;
      }
      p = static_cast<float*>(addr);
      cache[dev].store(p, std::memory_order_release);
    }
  }
  *out = p;
  return cudaSuccess;
}

}  // namespace

extern "C" {

int bc_decode_static_scratch(const bc_shape* s, const void* q, const void* k, const void* v,
                             const int* pages, const int* lengths, float* output, int splits,
                             void* stream) {
  if (!basic_shape_ok(s) || splits < 1 || splits > BC_MAX_SPLITS || !q || !k || !v || !pages ||
      !lengths || !output)
    return cudaErrorInvalidValue;
  const long long rows = (long long)s->batch * s->query_heads;
  const long long need = (long long)splits * rows * (s->dim + 2);
  if (need > BC_STATIC_SCRATCH_FLOATS) return cudaErrorInvalidValue;  // beyond the fixed array
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  float* scratch = nullptr;
  const cudaError_t e = static_scratch_address(dev, &scratch);
  if (e != cudaSuccess) return e;
  float* partial_a = scratch;                                  // splits * rows * dim
  float* partial_ml = scratch + (long long)splits * rows * s->dim;  // splits * rows * 2
  return paged_decode_core(s, q, k, v, pages, lengths, output, false,
                           1.0f / std::sqrt(float(s->dim)), splits,
                           splits > 1 ? kSplitGlobal : kSplitNone, false, partial_a, partial_ml,
                           false, nullptr, static_cast<cudaStream_t>(stream));
}

// ---------------------------------------------------------------------------
// Prompts and beams (bc_append.cuh, bc_chunk.cuh, bc_beam.cuh).
// ---------------------------------------------------------------------------
}  // extern "C"

namespace {

// One launch as a programmatic dependent of the kernel before it.
template <typename... P, typename... A>
cudaError_t launch_dependent(void (*kern)(P...), dim3 grid, int threads, size_t smem,
                             cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}

// Raises a kernel's dynamic shared memory limit once per device.
template <typename K>
cudaError_t raise_smem(K kern, size_t bytes, std::atomic<uint64_t>& configured, int dev) {
  if (configured.load(std::memory_order_relaxed) & (uint64_t(1) << dev)) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  if (e == cudaSuccess) configured.fetch_or(uint64_t(1) << dev);
  return e;
}

uintptr_t address_bits() { return 0; }
template <typename T, typename... R>
uintptr_t address_bits(const T* p, R... rest) {
  return reinterpret_cast<uintptr_t>(p) | address_bits(rest...);
}

// A cache whose rows the kernels may copy in 16-byte pieces.
bool layout_ok(const bc_kv_layout* l, int pages) {
  return l && (l->block_stride > 0 || pages == 1) && l->slot_stride > 0 && l->head_stride > 0 &&
         ((l->block_stride | l->slot_stride | l->head_stride) & 7) == 0;
}

// Pages whose slots an int can number.
bool pool_ok(int pages) { return pages >= 1 && pages <= 0x7fffffff / kPageSize; }

bool encode_map_n(CUtensorMap* map, int dtype, int rank, const void* base, const uint64_t* dims,
                  const uint64_t* strides_bytes, const uint32_t* box) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t gdim[5], gstr[4];
  cuuint32_t bdim[5], estr[5];
  for (int i = 0; i < rank; ++i) {
    gdim[i] = dims[i];
    bdim[i] = box[i];
    estr[i] = 1;
    if (i + 1 < rank) {
      if (strides_bytes[i] % 16 || strides_bytes[i] >= (uint64_t(1) << 40)) return false;
      gstr[i] = strides_bytes[i];
    }
  }
  return fn(map, dtype == BC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            cuuint32_t(rank), const_cast<void*>(base), gdim, gstr, bdim, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Q [tokens, heads, dim] as (dim, heads, tokens): boxes of one KV head's query
// heads of a row tile's tokens, 64 dims wide.
bool encode_rows_map(CUtensorMap* map, int dtype, const void* q, int dim, int heads, int tokens,
                     long long token_stride, int group, int tile_tokens) {
  const uint64_t dims[3] = {uint64_t(dim), uint64_t(heads), uint64_t(tokens)};
  // (one token: any valid stride)
  const uint64_t st[2] = {uint64_t(dim) * 2,
                          uint64_t(tokens > 1 ? token_stride : (long long)heads * dim) * 2};
  const uint32_t box[3] = {64, uint32_t(group), uint32_t(tile_tokens)};
  return st[1] > 0 && encode_map_n(map, dtype, 3, q, dims, st, box);
}

// K or V of a paged cache as (64 dims, 8 slots, 64-dim blocks of the heads, 2
// halves of a page, pages): a box is one head's 16 rows of a page, each half
// page a run of 8-row groups of its 64-dim blocks.
bool encode_pages_map(CUtensorMap* map, int dtype, const void* base, const bc_shape* s,
                      const bc_kv_layout* l) {
  const int kb = s->dim / 64;
  const uint64_t dims[5] = {64, 8, uint64_t((s->kv_heads - 1) * (l->head_stride / 64) + kb), 2,
                            uint64_t(s->physical_pages)};
  const uint64_t block = uint64_t(s->physical_pages > 1 ? l->block_stride : 16 * l->slot_stride);
  const uint64_t st[4] = {uint64_t(l->slot_stride) * 2, 128, uint64_t(l->slot_stride) * 16, block * 2};
  const uint32_t box[5] = {64, 8, uint32_t(kb), 2, 1};
  return encode_map_n(map, dtype, 5, base, dims, st, box);
}

bool chunk_shape_ok(const bc_shape* s) {
  // (a row's end, rounded up to a key tile, is an int too)
  return basic_shape_ok(s) && pool_ok(s->physical_pages) &&
         s->max_pages <= (0x7fffffff - kChTile) / kPageSize &&
         s->batch <= kChMaxBatch && s->query_heads / s->kv_heads <= 128;
}

// The launch of a chunk attention, from host-known bounds alone.
struct ChunkPlan {
  int blocks;    // thread blocks: one per SM, no more than there can be key tiles
  int rows;      // rows of a partial state
  size_t bytes;  // workspace; 0 where no item is long enough to be split
  ChunkPlan(const bc_shape* s, int tokens, int dev) {
    const int group = s->query_heads / s->kv_heads, tile = 128 / group;
    const long long key_tiles = (s->max_pages + kChTile / kPageSize - 1) / (kChTile / kPageSize);
    const long long items = ((long long)tokens / (2 * tile) + std::min(s->batch, tokens)) * s->kv_heads;
    blocks = int(std::min<long long>(std::min(dev < 0 ? 148 : sm_count(dev), 160), items * key_tiles));
    rows = tokens <= tile ? (tokens * group + 31) / 32 * 32 : 256;
    bytes = key_tiles <= kChWhole
                ? 0
                : size_t(blocks) * (2 * size_t(rows) * (s->dim * 4 + 8) + 32);
  }
};

// tanh(u) / u in powers of u^2 up to |u| = kTanhNear, fitted for the smallest largest
// error of tanh there: 1.2e-8 with these coefficients.
constexpr double kTanh[5] = {1.0, -0.33332759141921997, 0.13317517936229706, -0.05250634625554085,
                             0.016171788796782494};
constexpr double kTanhNear = 0.55;

ChunkCap chunk_cap(double scale, double softcap) {
  const double u = scale / softcap;  // of a score of 1
  const bool fold = u > 1e-4 && u < 1e4 && scale > 1e-5 && scale < 1e5;
  // (a cap beyond 2^126 caps no score, and with such a u a score is 0 or at the cap: both
  // stay within 32 bits)
  const double most = 8.5e37, cap = std::min(softcap, most), log2e = 1.4426950408889634;
  const double x = fold ? u : 1.0;
  ChunkCap c;
  double power = (fold ? scale : cap) * log2e;
  for (int i = 0; i < 5; ++i, power *= x * x) c.k[i] = float(kTanh[i] * power);
  c.near = float(kTanhNear / x);
  c.arg = float(2.0 * log2e * x);
  c.log2 = float(cap * log2e);
  c.pre = fold ? 1.f : float(std::min(scale / cap, most));
  return c;
}

template <int D, typename T, int MOD, bool F32>
cudaError_t launch_chunk_mod(ChunkParams& p, const CUtensorMap* maps, const ChunkPlan& plan,
                             int dev, cudaStream_t stream) {
  auto kern = chunk_mma_kernel<D, T, MOD, F32>;
  static std::atomic<size_t> smem_of[kMaxDevices];
  size_t smem = smem_of[dev].load(std::memory_order_relaxed);
  if (!smem) {
    // As for the tree kernel: the register split needs the launch budget.
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    if (fa.numRegs != kChLaunchRegs) return cudaErrorInvalidDeviceFunction;
    smem = ChunkGeom<D>::smem_bytes(fa.sharedSizeBytes);
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    smem_of[dev].store(smem, std::memory_order_relaxed);
  }
  p.smem_bytes = unsigned(smem);
  cudaError_t e = launch_dependent(kern, dim3(unsigned(plan.blocks)), kChThreads, smem, stream, p,
                                   maps[0], maps[1], maps[2]);
  if (e != cudaSuccess || plan.bytes == 0) return e;
  return launch_dependent(chunk_merge_kernel<D, T>,
                          dim3(unsigned(plan.blocks), unsigned((plan.rows + 31) / 32)),
                          kChMergeThreads, 0,
                          stream, p);
}

template <int D, typename T, bool F32>
cudaError_t launch_chunk_out(ChunkParams& p, const CUtensorMap* maps, const ChunkPlan& plan,
                         const bc_chunk_options* o, int dev, cudaStream_t stream) {
  switch ((o->softcap > 0.f ? 1 : 0) | (o->alibi_slopes ? 2 : 0)) {
    case 0: return launch_chunk_mod<D, T, 0, F32>(p, maps, plan, dev, stream);
    case 1: return launch_chunk_mod<D, T, 1, F32>(p, maps, plan, dev, stream);
    case 2: return launch_chunk_mod<D, T, 2, F32>(p, maps, plan, dev, stream);
    default: return launch_chunk_mod<D, T, 3, F32>(p, maps, plan, dev, stream);
  }
}

template <int D, typename T>
cudaError_t launch_chunk(ChunkParams& p, const CUtensorMap* maps, const ChunkPlan& plan,
                         const bc_chunk_options* o, int dev, cudaStream_t stream) {
  return p.out_f32 ? launch_chunk_out<D, T, true>(p, maps, plan, o, dev, stream)
                   : launch_chunk_out<D, T, false>(p, maps, plan, o, dev, stream);
}

// Rows are cut into the number of segments that takes the least time by count:
// waves of four blocks a SM times a segment's steps and its fixed work (the bound,
// the second look and the ranking, some six steps' time).
struct BeamPlan {
  int segments, segment;
  BeamPlan(int rows, int vocab, int type_bytes, int dev) {
    const int tile = beam_tile(type_bytes);
    const int steps = (vocab + tile - 1) / tile;
    const long long slots = 4ll * (dev < 0 ? 148 : sm_count(dev));
    long long least = -1;
    int per = steps;
    for (int s = 1; s <= steps && (s == 1 || (long long)rows * s <= 4 * slots); ++s) {
      const int each = (steps + s - 1) / s;
      const long long time = (((long long)rows * s + slots - 1) / slots) * (each + 6);
      if (least < 0 || time < least) {
        least = time;
        per = each;
      }
    }
    segment = per * tile;
    segments = (vocab + segment - 1) / segment;
  }
};

template <typename T>
cudaError_t launch_beam_segments(const BeamSelectParams& p, int dev, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};
  const cudaError_t e = raise_smem(beam_segment_kernel<T>, beam_smem(kBeamMaxK), configured, dev);
  if (e != cudaSuccess) return e;
  return launch_dependent(beam_segment_kernel<T>, dim3(unsigned(p.batch) * p.beams * p.segments),
                          kBeamThreads, beam_smem(p.k), stream, p);
}

int beam_type_bytes(int dtype) {
  return dtype == BC_F32 ? 4 : dtype == BC_F16 || dtype == BC_BF16 ? 2 : 0;
}

size_t beam_merge_smem(long long lists, int k) {
  return size_t(lists) * 8 + size_t((lists + 1) / 2) * 8 + size_t(k) * k * 12;
}

bool beam_shape_ok(int batch, int beams, int vocab, int k) {
  return batch >= 1 && beams >= 1 && beams <= kBeamMax && vocab >= 1 && vocab <= kBeamMaxVocab &&
         k >= 1 && k <= kBeamMaxK && k <= (long long)beams * vocab &&
         (long long)batch * beams <= 0xffffff;
}

bool reorder_shape_ok(int batch, int beams_in, int max_pages) {
  return batch >= 1 && beams_in >= 1 && beams_in <= kBeamMax && max_pages >= 1 &&
         max_pages <= 0x7fffffff / kPageSize &&
         (long long)batch * beams_in * ((max_pages + 31) / 32) * 32 <= 0x7fffffff;
}

}  // namespace

extern "C" {

int bc_append_plan(int batch, int physical_pages, const int* pages_in, int max_pages_in,
                   const int* lengths_in, const int* new_tokens, const int* refcount_in,
                   const int* free_stack_in, const int* free_count_in, int* refcount,
                   int* free_stack, int* free_count, int* pages_out, int max_pages_out,
                   int* lengths_out, int max_tokens, int* query_start, int* slot_map,
                   int* positions, int* clones, int* counts, int* scratch, void* stream) {
  if (batch < 1 || batch > BC_MAX_SEQUENCES || !pool_ok(physical_pages) || !pool_ok(max_pages_in) ||
      !pool_ok(max_pages_out) || max_tokens < 0 || !pages_in || !lengths_in || !new_tokens ||
      !refcount_in || !free_stack_in || !free_count_in || !refcount || !free_stack ||
      !free_count || !pages_out || !lengths_out || !query_start || !clones || !counts ||
      !scratch || (max_tokens > 0 && (!slot_map || !positions)) ||
      (pages_out == pages_in && max_pages_out != max_pages_in))
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  static std::atomic<uint64_t> configured{0};
  cudaError_t e =
      raise_smem(append_plan_kernel, append_plan_smem_bytes(BC_MAX_SEQUENCES), configured, dev);
  if (e != cudaSuccess) return e;
  const AppendPlanParams p{batch, physical_pages, max_pages_in, max_pages_out, max_tokens,
                           pages_in, lengths_in, new_tokens, refcount_in, free_stack_in,
                           free_count_in, refcount, free_stack, free_count, pages_out,
                           lengths_out, query_start, slot_map, positions, clones, counts,
                           scratch};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool copy = refcount != refcount_in || free_stack != free_stack_in;
  const int copiers = copy ? std::min(64, (physical_pages + 4 * kPlanThreads - 1) / (4 * kPlanThreads)) : 0;
  e = launch_dependent(append_plan_kernel, dim3(unsigned(1 + copiers)), kPlanThreads,
                       append_plan_smem_bytes(batch), st, p);
  if (e != cudaSuccess) return e;
  const int rows = kExpandThreads / 32;
  const int row_blocks = (batch + rows - 1) / rows;
  const int token_blocks = (max_tokens + kExpandTokens - 1) / kExpandTokens;
  return launch_dependent(append_expand_kernel, dim3(unsigned(row_blocks + token_blocks)),
                          kExpandThreads, 0, st, p, row_blocks);
}

int bc_append_kv(const bc_shape* s, int tokens, const void* k, long long k_stride, const void* v,
                 long long v_stride, void* cache_k, void* cache_v, const bc_kv_layout* layout,
                 const int* slot_map, const int* clones, int max_clones, const int* counts,
                 void* stream) {
  if (!s || s->kv_heads < 1 || (s->dim != 64 && s->dim != 128) || !pool_ok(s->physical_pages) ||
      tokens < 0 || !cache_k || !cache_v || !layout_ok(layout, s->physical_pages) || max_clones < 0 ||
      (tokens > 0 && (!k || !v || !slot_map)) || (max_clones > 0 && (!clones || !counts)) ||
      (address_bits(k, v, cache_k, cache_v) % 16) || ((k_stride | v_stride) & 7) ||
      k_stride < 0 || v_stride < 0 || (long long)s->kv_heads * s->dim > 0x7fffff)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  if (tokens == 0 && max_clones == 0) return cudaSuccess;
  AppendKvParams p = {};
  p.tokens = tokens;
  p.head_vecs = s->dim / 8;
  p.row_vecs = s->kv_heads * p.head_vecs;
  p.physical_pages = s->physical_pages;
  p.max_clones = max_clones;
  p.k = static_cast<const uint4*>(k);
  p.v = static_cast<const uint4*>(v);
  p.k_stride = k_stride / 8;
  p.v_stride = v_stride / 8;
  p.cache_k = static_cast<uint4*>(cache_k);
  p.cache_v = static_cast<uint4*>(cache_v);
  p.block_stride = layout->block_stride / 8;
  p.slot_stride = layout->slot_stride / 8;
  p.head_stride = layout->head_stride / 8;
  p.slot_map = slot_map;
  p.clones = clones;
  p.counts = counts;
  p.err = err;
  const int per_block = std::max(1, kAppendVecs * kAppendThreads / p.row_vecs);
  const int token_blocks = (tokens + per_block - 1) / per_block;
  return launch_dependent(append_kv_kernel, dim3(unsigned(token_blocks + max_clones), 2),
                          kAppendThreads, 0, static_cast<cudaStream_t>(stream), p, token_blocks,
                          per_block);
}

size_t bc_chunk_workspace_bytes(const bc_shape* s, int tokens) {
  if (!chunk_shape_ok(s) || tokens < 1) return 0;
  return ChunkPlan(s, tokens, current_device()).bytes;
}

int bc_chunk_attention(const bc_shape* s, int tokens, int dtype, const void* q,
                       long long q_stride, const void* k, const void* v,
                       const bc_kv_layout* layout, const int* pages, const int* query_start,
                       const int* lengths, const bc_chunk_options* options, void* output,
                       int output_f32, void* workspace, size_t workspace_bytes, void* stream) {
  if (!chunk_shape_ok(s) || tokens < 0 || (dtype != BC_F16 && dtype != BC_BF16) || !q || !k ||
      !v || !layout_ok(layout, s->physical_pages) || layout->head_stride % 64 || !pages ||
      !query_start || !lengths || !options || !output || (address_bits(q, k, v) % 16) ||
      address_bits(output) % 32 ||
      (q_stride & 7) || q_stride < 0 || !(options->scale > 0.f) || std::isinf(options->scale) ||
      !(options->softcap >= 0.f) || std::isinf(options->softcap) || options->window < 0)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  const ChunkPlan plan(s, std::max(tokens, 1), dev);
  if (workspace_bytes < plan.bytes ||
      (plan.bytes > 0 && (!workspace || address_bits(workspace) % 16)))
    return cudaErrorInvalidValue;
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  if (tokens == 0) return cudaSuccess;
  ChunkParams p = {};
  p.batch = s->batch;
  p.tokens = tokens;
  p.hq = s->query_heads;
  p.hkv = s->kv_heads;
  p.group = s->query_heads / s->kv_heads;
  p.tile_tokens = 128 / p.group;
  p.max_pages = s->max_pages;
  p.physical_pages = s->physical_pages;
  // (a window as wide as the table hides nothing)
  p.window = options->window < s->max_pages * kPageSize ? options->window : 0;
  p.head_blocks = int(layout->head_stride / 64);
  p.pages = pages;
  p.query_start = query_start;
  p.lengths = lengths;
  p.prefix = options->prefix;
  p.key_start = options->key_start;
  p.slopes = options->alibi_slopes;
  p.out = output;
  p.out_f32 = output_f32;
  p.scale_log2 = options->scale * kLog2e;
  if (options->softcap > 0.f) p.cap = chunk_cap(options->scale, options->softcap);
  p.part_rows = plan.rows;
  if (plan.bytes > 0) {
    p.part_o = static_cast<float4*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + size_t(plan.blocks) * 2 * plan.rows * (s->dim / 4));
    p.sched = reinterpret_cast<int*>(p.part_ml + size_t(plan.blocks) * 2 * plan.rows);
  }
  p.err = err;
  p.token = next_launch_token();
  CUtensorMap maps[3];
  if (!encode_rows_map(&maps[0], dtype, q, s->dim, s->query_heads, tokens, q_stride, p.group,
                       p.tile_tokens) ||
      !encode_pages_map(&maps[1], dtype, k, s, layout) ||
      !encode_pages_map(&maps[2], dtype, v, s, layout))
    return cudaErrorInvalidValue;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s->dim == 64)
    return dtype == BC_F16 ? launch_chunk<64, __half>(p, maps, plan, options, dev, st)
                           : launch_chunk<64, __nv_bfloat16>(p, maps, plan, options, dev, st);
  return dtype == BC_F16 ? launch_chunk<128, __half>(p, maps, plan, options, dev, st)
                         : launch_chunk<128, __nv_bfloat16>(p, maps, plan, options, dev, st);
}

size_t bc_beam_workspace_bytes(int batch, int beams, int vocab, int k, int dtype) {
  if (!beam_shape_ok(batch, beams, vocab, k) || beam_type_bytes(dtype) == 0) return 0;
  // per segment: k keys, its sum and its largest logit
  const BeamPlan plan(batch * beams, vocab, beam_type_bytes(dtype), current_device());
  return size_t(batch) * beams * plan.segments * (size_t(k) * 8 + 8 + 4);
}

int bc_beam_select(int batch, int beams, int vocab, int k, int dtype, const void* logits,
                   long long row_stride, const float* scores, float* out_scores, int* out_tokens,
                   int* out_parents, void* workspace, size_t workspace_bytes, void* stream) {
  if (!beam_shape_ok(batch, beams, vocab, k) ||
      beam_type_bytes(dtype) == 0 || !logits || row_stride < vocab ||
      !scores || !out_scores || !out_tokens || !out_parents || !workspace ||
      address_bits(workspace) % 16 ||
      address_bits(logits) % beam_type_bytes(dtype) ||
      workspace_bytes < bc_beam_workspace_bytes(batch, beams, vocab, k, dtype))
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  BeamSelectParams p = {};
  p.batch = batch;
  p.beams = beams;
  p.vocab = vocab;
  p.k = k;
  const BeamPlan plan(batch * beams, vocab, beam_type_bytes(dtype), dev);
  p.segments = plan.segments;
  p.segment = plan.segment;
  p.logits = logits;
  p.row_stride = row_stride;
  p.scores = scores;
  p.out_scores = out_scores;
  p.out_tokens = out_tokens;
  p.out_parents = out_parents;
  const size_t lists = size_t(batch) * beams * p.segments;
  p.keys = static_cast<unsigned long long*>(workspace);
  p.seg_sum = reinterpret_cast<double*>(p.keys + lists * k);
  p.seg_max = reinterpret_cast<float*>(p.seg_sum + lists);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = dtype == BC_F16    ? launch_beam_segments<__half>(p, dev, st)
                  : dtype == BC_BF16 ? launch_beam_segments<__nv_bfloat16>(p, dev, st)
                                     : launch_beam_segments<float>(p, dev, st);
  if (e != cudaSuccess) return e;
  static std::atomic<uint64_t> configured{0};
  // (a request's lists: at most sixteen blocks a SM, or one a beam)
  e = raise_smem(beam_merge_kernel, beam_merge_smem(std::max(16 * sm_count(dev), kBeamMax), kBeamMaxK),
                 configured, dev);
  if (e != cudaSuccess) return e;
  return launch_dependent(beam_merge_kernel, dim3(unsigned(batch)), kBeamMergeThreads,
                          beam_merge_smem((long long)beams * p.segments, k), st, p);
}

size_t bc_reorder_workspace_bytes(int batch, int beams_in, int max_pages) {
  if (!reorder_shape_ok(batch, beams_in, max_pages)) return 0;
  return size_t(batch) * beams_in * ((max_pages + 31) / 32) * 4;
}

int bc_beam_reorder(int batch, int beams_in, int beams_out, int physical_pages,
                    const int* pages_in, int max_pages, const int* lengths_in,
                    const int* parents, const int* refcount_in, const int* free_stack_in,
                    const int* free_count_in, int* refcount, int* free_stack, int* free_count,
                    int* pages_out, int* lengths_out, void* workspace, size_t workspace_bytes,
                    void* stream) {
  if (!reorder_shape_ok(batch, beams_in, max_pages) || beams_out < 1 || beams_out > kBeamMax ||
      !pool_ok(physical_pages) || !pages_in || !lengths_in || !parents || !refcount_in ||
      !free_stack_in || !free_count_in || !refcount || !free_stack || !free_count || !pages_out ||
      !lengths_out || pages_out == pages_in || lengths_out == lengths_in || !workspace ||
      address_bits(workspace) % 4 ||
      workspace_bytes < bc_reorder_workspace_bytes(batch, beams_in, max_pages))
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  BeamReorderParams p = {};
  p.batch = batch;
  p.beams_in = beams_in;
  p.beams_out = beams_out;
  p.max_pages = max_pages;
  p.physical_pages = physical_pages;
  p.words = (max_pages + 31) / 32;
  p.parents = parents;
  p.pages_in = pages_in;
  p.lengths_in = lengths_in;
  p.refcount_in = refcount_in;
  p.free_stack_in = free_stack_in;
  p.free_count_in = free_count_in;
  p.refcount = refcount;
  p.free_stack = free_stack;
  p.free_count = free_count;
  p.pages_out = pages_out;
  p.lengths_out = lengths_out;
  p.marks = static_cast<unsigned*>(workspace);
  p.err = err;
  const int row_blocks = int(((long long)batch * p.words + kReorderWarps - 1) / kReorderWarps);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static std::atomic<uint64_t> configured{0};
  cudaError_t e = raise_smem(beam_release_kernel, kReleaseSmem, configured, dev);
  if (e == cudaSuccess && (refcount != refcount_in || free_stack != free_stack_in))
    e = launch_dependent(pool_copy_kernel, dim3(unsigned(std::min(256, (physical_pages + 255) / 256))),
                         256, 0, st, physical_pages, refcount_in, refcount, free_stack_in, free_stack);
  if (e == cudaSuccess)
    e = launch_dependent(beam_rows_kernel, dim3(unsigned(row_blocks)), kReorderWarps * 32, 0, st, p);
  if (e != cudaSuccess) return e;
  return launch_dependent(beam_release_kernel, dim3(1), kReleaseThreads, kReleaseSmem, st, p);
}

int bc_selftest_bounded_wait(int ctas, int smem_bytes, unsigned limit_us, void* stream) {
  if (ctas < 1 || smem_bytes < 0 || smem_bytes > 200 * 1024 || limit_us < 1 ||
      limit_us > 2000000u)
    return cudaErrorInvalidValue;
  const int dev = current_device();
  if (dev < 0) return cudaErrorInvalidDevice;
  unsigned* err = error_word(dev);
  if (!err) return cudaErrorInvalidDevice;
  cudaError_t e = cudaFuncSetAttribute(selftest_wait_kernel,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
  if (e != cudaSuccess) return e;
  selftest_wait_kernel<<<ctas, 32, size_t(smem_bytes), static_cast<cudaStream_t>(stream)>>>(
      (unsigned long long)limit_us * 1000ull, next_launch_token(), err);
  return cudaGetLastError();
}

unsigned bc_last_device_error(int reset) {
  const int dev = current_device();
  if (dev < 0) return 0xffffffffu;
  if (cudaDeviceSynchronize() != cudaSuccess) return 0xffffffffu;
  unsigned word = 0;
  if (cudaMemcpyFromSymbol(&word, g_error_word, sizeof(word)) != cudaSuccess) return 0xffffffffu;
  if (reset) {
    // (the abort token too: a captured graph keeps its launches' tokens, so
    // a replay after a timeout would otherwise find itself aborted)
    const unsigned zero = 0;
    if (cudaMemcpyToSymbol(g_error_word, &zero, sizeof(zero)) != cudaSuccess ||
        cudaMemcpyToSymbol(g_abort_token, &zero, sizeof(zero)) != cudaSuccess)
      return 0xffffffffu;
  }
  return word;
}

const char* bc_version(void) { return "branchcraft-b200 0.1.0 (sm_100a)"; }

}  // extern "C"
