// PyTorch dispatcher binding: TORCH_LIBRARY(branchcraft) with the reference's
// three schemas (bindings/torch_ops.cpp:144-148) and the same argument checks
// (bindings/torch_ops.cpp:11-140), plus the ops the reference lacks:
//   paged_decode          paged GQA decode, FP32 out (optional split count)
//   tree_verify_out       tree verify into a preallocated FP32 or FP16 output
//   packed_decode_kv_out  decode from separate K / V views of one packed cache
//                         (vLLM's [num_blocks, 2, 16, Hkv, D]: k = cache[:, 0])
//   commit_batch_         a whole batch of copy-on-write commits
//   append_plan(_)        page tables, slot map and positions of new tokens
//   append_kv_            their K/V rows (and page clones) into the paged cache
//   chunk_attention(_out) attention of a chunk of new tokens over that cache
//   beam_select           the best (beam, token) pairs of every request
//   beam_reorder(_)       page tables after the beams' new parents
// Every op calls the C ABI (branchcraft.h) on the current CUDA stream.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "branchcraft.h"

namespace {

void check_cuda_contiguous(const at::Tensor& t, const char* name, at::ScalarType dtype) {
  TORCH_CHECK(t.is_cuda(), name, " must be CUDA");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.scalar_type() == dtype, name, " has wrong dtype");
}

void check_launch(int err, const char* op) {
  TORCH_CHECK(err == 0, op, ": ", cudaGetErrorString(static_cast<cudaError_t>(err)));
}

void* stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_tree(const at::Tensor& q, const at::Tensor& prefix_k, const at::Tensor& prefix_v,
                const at::Tensor& pages, const at::Tensor& lengths, const at::Tensor& draft_k,
                const at::Tensor& draft_v, const at::Tensor& parent) {
  check_cuda_contiguous(q, "q", at::kHalf);
  check_cuda_contiguous(prefix_k, "prefix_k", at::kHalf);
  check_cuda_contiguous(prefix_v, "prefix_v", at::kHalf);
  check_cuda_contiguous(draft_k, "draft_k", at::kHalf);
  check_cuda_contiguous(draft_v, "draft_v", at::kHalf);
  check_cuda_contiguous(pages, "pages", at::kInt);
  check_cuda_contiguous(lengths, "lengths", at::kInt);
  check_cuda_contiguous(parent, "parent", at::kInt);
  TORCH_CHECK(q.dim() == 4 && prefix_k.dim() == 4 && prefix_v.dim() == 4 && draft_k.dim() == 4 &&
                  draft_v.dim() == 4 && pages.dim() == 2 && lengths.dim() == 1 &&
                  parent.dim() == 2,
              "invalid tree tensor rank");
  const int64_t b = q.size(0), nodes = q.size(1), hq = q.size(2), d = q.size(3);
  const int64_t hkv = prefix_k.size(2);
  TORCH_CHECK(b > 0 && nodes > 0 && nodes <= BC_MAX_NODES && hq > 0 && hkv > 0 && hq % hkv == 0 &&
                  (d == 64 || d == 128),
              "unsupported tree shape");
  TORCH_CHECK(prefix_k.size(1) == BC_PAGE_SIZE && prefix_k.size(3) == d &&
                  prefix_v.sizes() == prefix_k.sizes(),
              "prefix K/V shape mismatch");
  TORCH_CHECK(draft_k.sizes() == at::IntArrayRef({b, nodes, hkv, d}) &&
                  draft_v.sizes() == draft_k.sizes(),
              "draft K/V shape mismatch");
  TORCH_CHECK(pages.size(0) == b && lengths.size(0) == b &&
                  parent.sizes() == at::IntArrayRef({b, nodes}),
              "tree metadata shape mismatch");
  TORCH_CHECK(q.device() == prefix_k.device() && q.device() == prefix_v.device() &&
                  q.device() == draft_k.device() && q.device() == draft_v.device() &&
                  q.device() == pages.device() && q.device() == lengths.device() &&
                  q.device() == parent.device(),
              "all tensors must share a device");
}

int launch_tree(const at::Tensor& q, const at::Tensor& prefix_k, const at::Tensor& prefix_v,
                const at::Tensor& pages, const at::Tensor& lengths, const at::Tensor& draft_k,
                const at::Tensor& draft_v, const at::Tensor& parent, at::Tensor& output) {
  const bc_shape s{int(q.size(0)), int(q.size(2)), int(prefix_k.size(2)), int(q.size(3)),
                   int(pages.size(1)), int(prefix_k.size(0))};
  const int nodes = int(q.size(1));
  if (output.scalar_type() == at::kHalf)
    return bc_tree_verify_f16(&s, q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(),
                              pages.data_ptr<int>(), lengths.data_ptr<int>(), draft_k.data_ptr(),
                              draft_v.data_ptr(), parent.data_ptr<int>(), output.data_ptr(),
                              nodes, stream());
  return bc_tree_verify(&s, q.data_ptr(), prefix_k.data_ptr(), prefix_v.data_ptr(),
                        pages.data_ptr<int>(), lengths.data_ptr<int>(), draft_k.data_ptr(),
                        draft_v.data_ptr(), parent.data_ptr<int>(), output.data_ptr<float>(),
                        nodes, stream());
}

at::Tensor tree_verify_cuda(const at::Tensor& q, const at::Tensor& prefix_k,
                            const at::Tensor& prefix_v, const at::Tensor& pages,
                            const at::Tensor& lengths, const at::Tensor& draft_k,
                            const at::Tensor& draft_v, const at::Tensor& parent) {
  check_tree(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent);
  auto output = at::empty(q.sizes(), q.options().dtype(at::kFloat));
  check_launch(launch_tree(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent, output),
               "tree_verify");
  return output;
}

at::Tensor& tree_verify_out_cuda(const at::Tensor& q, const at::Tensor& prefix_k,
                                 const at::Tensor& prefix_v, const at::Tensor& pages,
                                 const at::Tensor& lengths, const at::Tensor& draft_k,
                                 const at::Tensor& draft_v, const at::Tensor& parent,
                                 at::Tensor& output) {
  check_tree(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent);
  TORCH_CHECK(output.is_cuda() && output.is_contiguous() && output.sizes() == q.sizes() &&
                  (output.scalar_type() == at::kFloat || output.scalar_type() == at::kHalf) &&
                  output.device() == q.device(),
              "output must be a contiguous CUDA FP32/FP16 tensor shaped like q");
  check_launch(launch_tree(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent, output),
               "tree_verify_out");
  return output;
}

void check_packed_common(const at::Tensor& q, const at::Tensor& pages, const at::Tensor& lengths,
                         const at::Tensor& output) {
  check_cuda_contiguous(q, "q", at::kHalf);
  check_cuda_contiguous(pages, "pages", at::kInt);
  check_cuda_contiguous(lengths, "lengths", at::kInt);
  check_cuda_contiguous(output, "output", at::kHalf);
  TORCH_CHECK(q.dim() == 3 && pages.dim() == 2 && lengths.dim() == 1,
              "invalid packed decode tensor rank");
}

at::Tensor& packed_decode_out_cuda(const at::Tensor& q, const at::Tensor& packed_kv,
                                   const at::Tensor& pages, const at::Tensor& lengths,
                                   at::Tensor& output, double scale) {
  check_packed_common(q, pages, lengths, output);
  TORCH_CHECK(packed_kv.is_cuda() && packed_kv.scalar_type() == at::kHalf &&
                  packed_kv.dim() == 4 && packed_kv.stride(3) == 1,
              "packed_kv must be a CUDA FP16 tensor with contiguous content dim");
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2);
  const int64_t hkv = packed_kv.size(1);
  TORCH_CHECK(b > 0 && hq > 0 && hkv > 0 && hq % hkv == 0 && (d == 64 || d == 128),
              "unsupported packed decode shape");
  TORCH_CHECK(packed_kv.size(2) == BC_PAGE_SIZE && packed_kv.size(3) == 2 * d,
              "packed KV shape mismatch");
  TORCH_CHECK(pages.size(0) == b && lengths.size(0) == b && output.numel() == q.numel(),
              "packed decode metadata/output mismatch");
  TORCH_CHECK(q.device() == packed_kv.device() && q.device() == pages.device() &&
                  q.device() == lengths.device() && q.device() == output.device(),
              "all tensors must share a device");
  const bc_shape s{int(b), int(hq), int(hkv), int(d), int(pages.size(1)), int(packed_kv.size(0))};
  check_launch(bc_packed_decode(&s, q.data_ptr(), packed_kv.data_ptr(), pages.data_ptr<int>(),
                                lengths.data_ptr<int>(), output.data_ptr(), packed_kv.stride(0),
                                packed_kv.stride(1), packed_kv.stride(2), float(scale), stream()),
               "packed_decode_out");
  return output;
}

at::Tensor& packed_decode_kv_out_cuda(const at::Tensor& q, const at::Tensor& k_cache,
                                      const at::Tensor& v_cache, const at::Tensor& pages,
                                      const at::Tensor& lengths, at::Tensor& output, double scale,
                                      int64_t splits) {
  check_packed_common(q, pages, lengths, output);
  TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_cache.scalar_type() == at::kHalf &&
                  v_cache.scalar_type() == at::kHalf && k_cache.dim() == 4 &&
                  v_cache.sizes() == k_cache.sizes() && k_cache.strides() == v_cache.strides() &&
                  k_cache.stride(3) == 1,
              "k_cache / v_cache must be FP16 CUDA views [P, Hkv, 16, D] with equal strides "
              "and a contiguous last dim");
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2);
  const int64_t hkv = k_cache.size(1);
  TORCH_CHECK(b > 0 && hq > 0 && hkv > 0 && hq % hkv == 0 && (d == 64 || d == 128),
              "unsupported packed decode shape");
  TORCH_CHECK(k_cache.size(2) == BC_PAGE_SIZE && k_cache.size(3) == d, "KV view shape mismatch");
  TORCH_CHECK(pages.size(0) == b && lengths.size(0) == b && output.numel() == q.numel(),
              "packed decode metadata/output mismatch");
  TORCH_CHECK(splits >= 0 && splits <= 8, "splits must be 0 (auto) or 1..8");
  const auto* kb = static_cast<const at::Half*>(k_cache.data_ptr());
  const auto* vb = static_cast<const at::Half*>(v_cache.data_ptr());
  const bc_shape s{int(b), int(hq), int(hkv), int(d), int(pages.size(1)), int(k_cache.size(0))};
  check_launch(bc_packed_decode_kv(&s, q.data_ptr(), kb, pages.data_ptr<int>(),
                                   lengths.data_ptr<int>(), output.data_ptr(), k_cache.stride(0),
                                   k_cache.stride(1), k_cache.stride(2), (long long)(vb - kb),
                                   float(scale), int(splits), stream()),
               "packed_decode_kv_out");
  return output;
}

at::Tensor paged_decode_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                             const at::Tensor& pages, const at::Tensor& lengths, int64_t splits) {
  check_cuda_contiguous(q, "q", at::kHalf);
  check_cuda_contiguous(k, "k", at::kHalf);
  check_cuda_contiguous(v, "v", at::kHalf);
  check_cuda_contiguous(pages, "pages", at::kInt);
  check_cuda_contiguous(lengths, "lengths", at::kInt);
  TORCH_CHECK(q.dim() == 3 && k.dim() == 4 && v.sizes() == k.sizes() && pages.dim() == 2 &&
                  lengths.dim() == 1,
              "invalid paged decode tensor rank");
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2), hkv = k.size(2);
  TORCH_CHECK(k.size(1) == BC_PAGE_SIZE && k.size(3) == d && hkv > 0 && hq % hkv == 0 &&
                  (d == 64 || d == 128) && pages.size(0) == b && lengths.size(0) == b,
              "paged decode shape mismatch");
  TORCH_CHECK(q.device() == k.device() && q.device() == v.device() &&
                  q.device() == pages.device() && q.device() == lengths.device(),
              "all tensors must share a device");
  TORCH_CHECK(splits >= 0 && splits <= BC_MAX_SPLITS, "splits must be 0 (auto) or 1..64");
  auto output = at::empty(q.sizes(), q.options().dtype(at::kFloat));
  const bc_shape s{int(b), int(hq), int(hkv), int(d), int(pages.size(1)), int(k.size(0))};
  if (splits > 8) {
    auto pa = at::empty({splits * b * hq * d}, q.options().dtype(at::kFloat));
    auto pml = at::empty({splits * b * hq * 2}, q.options().dtype(at::kFloat));
    check_launch(bc_decode(&s, q.data_ptr(), k.data_ptr(), v.data_ptr(), pages.data_ptr<int>(),
                           lengths.data_ptr<int>(), output.data_ptr<float>(),
                           pa.data_ptr<float>(), pml.data_ptr<float>(), int(splits), stream()),
                 "paged_decode");
  } else {
    check_launch(bc_paged_decode(&s, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                 pages.data_ptr<int>(), lengths.data_ptr<int>(),
                                 output.data_ptr<float>(), int(splits), stream()),
                 "paged_decode");
  }
  return output;
}

void commit_path_cuda(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& draft_k,
                      const at::Tensor& draft_v, const at::Tensor& path_nodes,
                      const at::Tensor& dest_pages, const at::Tensor& dest_slots,
                      int64_t request) {
  check_cuda_contiguous(cache_k, "cache_k", at::kHalf);
  check_cuda_contiguous(cache_v, "cache_v", at::kHalf);
  check_cuda_contiguous(draft_k, "draft_k", at::kHalf);
  check_cuda_contiguous(draft_v, "draft_v", at::kHalf);
  check_cuda_contiguous(path_nodes, "path_nodes", at::kInt);
  check_cuda_contiguous(dest_pages, "dest_pages", at::kInt);
  check_cuda_contiguous(dest_slots, "dest_slots", at::kInt);
  TORCH_CHECK(cache_k.dim() == 4 && cache_v.sizes() == cache_k.sizes() && draft_k.dim() == 4 &&
                  draft_v.sizes() == draft_k.sizes() && path_nodes.dim() == 1 &&
                  dest_pages.sizes() == path_nodes.sizes() &&
                  dest_slots.sizes() == path_nodes.sizes(),
              "commit tensor shape mismatch");
  const int64_t b = draft_k.size(0), nodes = draft_k.size(1), hkv = draft_k.size(2),
                d = draft_k.size(3);
  TORCH_CHECK(request >= 0 && request < b && path_nodes.numel() > 0 &&
                  path_nodes.numel() <= nodes && cache_k.size(1) == BC_PAGE_SIZE &&
                  cache_k.size(2) == hkv && cache_k.size(3) == d,
              "invalid commit destination");
  TORCH_CHECK(cache_k.device() == draft_k.device() && cache_k.device() == cache_v.device() &&
                  cache_k.device() == draft_v.device() &&
                  cache_k.device() == path_nodes.device() &&
                  cache_k.device() == dest_pages.device() &&
                  cache_k.device() == dest_slots.device(),
              "all tensors must share a device");
  const bc_shape s{int(b), int(hkv), int(hkv), int(d), 1, int(cache_k.size(0))};
  check_launch(bc_commit_path(&s, draft_k.data_ptr(), draft_v.data_ptr(), cache_k.data_ptr(),
                              cache_v.data_ptr(), path_nodes.data_ptr<int>(),
                              dest_pages.data_ptr<int>(), dest_slots.data_ptr<int>(),
                              int(request), int(nodes), int(path_nodes.numel()), stream()),
               "commit_path_");
}

void commit_batch_cuda(at::Tensor& cache_k, at::Tensor& cache_v, const at::Tensor& draft_k,
                       const at::Tensor& draft_v, const at::Tensor& clone_src,
                       const at::Tensor& clone_dst, const at::Tensor& entry_request,
                       const at::Tensor& entry_node, const at::Tensor& entry_page,
                       const at::Tensor& entry_slot) {
  check_cuda_contiguous(cache_k, "cache_k", at::kHalf);
  check_cuda_contiguous(cache_v, "cache_v", at::kHalf);
  check_cuda_contiguous(draft_k, "draft_k", at::kHalf);
  check_cuda_contiguous(draft_v, "draft_v", at::kHalf);
  for (const at::Tensor* t : {&clone_src, &clone_dst, &entry_request, &entry_node, &entry_page,
                              &entry_slot})
    check_cuda_contiguous(*t, "commit plan", at::kInt);
  TORCH_CHECK(cache_k.dim() == 4 && cache_v.sizes() == cache_k.sizes() && draft_k.dim() == 4 &&
                  draft_v.sizes() == draft_k.sizes() && clone_src.sizes() == clone_dst.sizes() &&
                  entry_node.sizes() == entry_request.sizes() &&
                  entry_page.sizes() == entry_request.sizes() &&
                  entry_slot.sizes() == entry_request.sizes(),
              "commit_batch_ tensor shape mismatch");
  const int64_t hkv = draft_k.size(2), d = draft_k.size(3);
  TORCH_CHECK(cache_k.size(1) == BC_PAGE_SIZE && cache_k.size(2) == hkv && cache_k.size(3) == d,
              "cache / draft head shape mismatch");
  const bc_shape s{int(draft_k.size(0)), int(hkv), int(hkv), int(d), 1, int(cache_k.size(0))};
  check_launch(bc_commit_batch(&s, int(draft_k.size(1)), draft_k.data_ptr(), draft_v.data_ptr(),
                               cache_k.data_ptr(), cache_v.data_ptr(),
                               clone_src.data_ptr<int>(), clone_dst.data_ptr<int>(),
                               int(clone_src.numel()), entry_request.data_ptr<int>(),
                               entry_node.data_ptr<int>(), entry_page.data_ptr<int>(),
                               entry_slot.data_ptr<int>(), int(entry_node.numel()), stream()),
               "commit_batch_");
}

// ------------------------------------------------------- prompts and beams
// These run on the device of their tensors, whichever is current.

using at::Tensor;

// (past the dispatcher: a step's small outputs cost the host more than the GPU)
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

void check_state(const Tensor& pages, const Tensor& lengths, const Tensor& refcount,
                 const Tensor& free_stack, const Tensor& free_count) {
  for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{pages, "pages"},
                                {lengths, "lengths"},
                                {refcount, "refcount"},
                                {free_stack, "free_stack"},
                                {free_count, "free_count"}}) {
    check_cuda_contiguous(t, name, at::kInt);
    TORCH_CHECK(t.device() == pages.device(), "all tensors must share a device");
  }
  TORCH_CHECK(refcount.dim() == 1 && refcount.numel() >= 1 &&
                  free_stack.sizes() == refcount.sizes() && free_count.numel() == 1,
              "the pool's state is refcount [P], free_stack [P], free_count [1]");
}

using PlanOutputs = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>;

PlanOutputs run_append_plan(const Tensor& pages, const Tensor& lengths, const Tensor& new_tokens,
                            const Tensor& refcount, const Tensor& free_stack,
                            const Tensor& free_count, Tensor pages_out, Tensor lengths_out,
                            Tensor refcount_out, Tensor free_stack_out, Tensor free_count_out,
                            int64_t max_tokens, const char* op) {
  const int64_t batch = pages.size(0);
  auto query_start = fresh({batch + 1}, at::kInt, pages);
  auto slot_map = fresh({max_tokens}, at::kInt, pages);
  auto positions = fresh({max_tokens}, at::kInt, pages);
  auto clones = fresh({3, batch}, at::kInt, pages);
  auto counts = fresh({3}, at::kInt, pages);
  auto scratch = fresh({batch + 1}, at::kInt, pages);
  check_launch(
      bc_append_plan(int(batch), int(refcount.numel()), pages.data_ptr<int>(), int(pages.size(1)),
                     lengths.data_ptr<int>(), new_tokens.data_ptr<int>(),
                     refcount.data_ptr<int>(), free_stack.data_ptr<int>(),
                     free_count.data_ptr<int>(), refcount_out.data_ptr<int>(),
                     free_stack_out.data_ptr<int>(), free_count_out.data_ptr<int>(),
                     pages_out.data_ptr<int>(), int(pages_out.size(1)),
                     lengths_out.data_ptr<int>(), int(max_tokens), query_start.data_ptr<int>(),
                     slot_map.data_ptr<int>(), positions.data_ptr<int>(), clones.data_ptr<int>(),
                     counts.data_ptr<int>(), scratch.data_ptr<int>(), stream()),
      op);
  return {query_start, slot_map, positions, clones, counts};
}

void check_append_plan(const Tensor& pages, const Tensor& lengths, const Tensor& new_tokens,
                       const Tensor& refcount, const Tensor& free_stack, const Tensor& free_count,
                       int64_t max_tokens, int64_t max_pages) {
  check_state(pages, lengths, refcount, free_stack, free_count);
  check_cuda_contiguous(new_tokens, "new_tokens", at::kInt);
  TORCH_CHECK(new_tokens.device() == pages.device(), "all tensors must share a device");
  TORCH_CHECK(pages.dim() == 2 && pages.size(0) >= 1 && pages.size(0) <= BC_MAX_SEQUENCES &&
                  pages.size(1) >= 1 && lengths.dim() == 1 && lengths.size(0) == pages.size(0) &&
                  new_tokens.sizes() == lengths.sizes(),
              "pages is [sequences, max_pages] (at most ", BC_MAX_SEQUENCES,
              " sequences), lengths and new_tokens [sequences]");
  TORCH_CHECK(max_tokens >= 0 && max_tokens <= INT32_MAX && max_pages >= 0 &&
                  max_pages <= INT32_MAX / BC_PAGE_SIZE,
              "max_tokens or max_pages out of range");
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>
append_plan_cuda(const Tensor& pages, const Tensor& lengths, const Tensor& new_tokens,
                 const Tensor& refcount, const Tensor& free_stack, const Tensor& free_count,
                 int64_t max_tokens, int64_t max_pages) {
  check_append_plan(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens,
                    max_pages);
  const c10::cuda::CUDAGuard guard(pages.device());
  auto pages_out =
      fresh({pages.size(0), max_pages > 0 ? max_pages : pages.size(1)}, at::kInt, pages);
  auto lengths_out = fresh(lengths.sizes(), at::kInt, pages),
       refcount_out = fresh(refcount.sizes(), at::kInt, pages),
       stack_out = fresh(free_stack.sizes(), at::kInt, pages),
       count_out = fresh(free_count.sizes(), at::kInt, pages);
  auto [qs, sm, pos, cl, cn] =
      run_append_plan(pages, lengths, new_tokens, refcount, free_stack, free_count, pages_out,
                      lengths_out, refcount_out, stack_out, count_out, max_tokens, "append_plan");
  return {pages_out, lengths_out, refcount_out, stack_out, count_out, qs, sm, pos, cl, cn};
}

PlanOutputs append_plan_inplace_cuda(Tensor& pages, Tensor& lengths, const Tensor& new_tokens,
                                     Tensor& refcount, const Tensor& free_stack,
                                     Tensor& free_count, int64_t max_tokens) {
  check_append_plan(pages, lengths, new_tokens, refcount, free_stack, free_count, max_tokens, 0);
  const c10::cuda::CUDAGuard guard(pages.device());
  return run_append_plan(pages, lengths, new_tokens, refcount, free_stack, free_count, pages,
                         lengths, refcount, free_stack, free_count, max_tokens, "append_plan_");
}

bool is_16bit(const Tensor& t) {
  return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16;
}

// K and V of a paged cache, [P, 16, Hkv, D] of equal strides.
bc_kv_layout check_cache(const Tensor& k, const Tensor& v) {
  TORCH_CHECK(k.is_cuda() && v.is_cuda() && is_16bit(k) && v.scalar_type() == k.scalar_type() &&
                  k.device() == v.device(),
              "K and V caches must be FP16 or BF16 on one CUDA device");
  TORCH_CHECK(k.dim() == 4 && k.size(0) >= 1 && k.size(1) == BC_PAGE_SIZE && k.size(2) >= 1 &&
                  (k.size(3) == 64 || k.size(3) == 128) && v.sizes() == k.sizes() &&
                  v.strides() == k.strides() && k.stride(3) == 1,
              "K and V caches must be [P, 16, Hkv, 64 or 128] with equal strides and a "
              "contiguous last dimension");
  return bc_kv_layout{k.stride(0), k.stride(1), k.size(2) > 1 ? k.stride(2) : k.size(3)};
}

// Elements between two tokens' rows of [tokens, heads, D] (one token: any).
int64_t token_stride(const Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2);
}

void append_kv_cuda(Tensor& cache_k, Tensor& cache_v, const Tensor& k, const Tensor& v,
                    const Tensor& slot_map, const std::optional<Tensor>& clones,
                    const std::optional<Tensor>& counts) {
  const bc_kv_layout layout = check_cache(cache_k, cache_v);
  check_cuda_contiguous(slot_map, "slot_map", at::kInt);
  const int64_t hkv = cache_k.size(2), d = cache_k.size(3);
  for (const Tensor* t : {&k, &v})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == cache_k.scalar_type() && t->dim() == 3 &&
                    t->size(0) == slot_map.numel() && t->size(1) == hkv && t->size(2) == d &&
                    t->stride(2) == 1 && (hkv == 1 || t->stride(1) == d),
                "k and v must be [tokens, Hkv, D] of the cache's type, each token's heads "
                "contiguous");
  TORCH_CHECK(slot_map.dim() == 1 && clones.has_value() == counts.has_value(),
              "slot_map is [tokens]; clones and counts go together");
  if (clones) {
    check_cuda_contiguous(*clones, "clones", at::kInt);
    check_cuda_contiguous(*counts, "counts", at::kInt);
    TORCH_CHECK(clones->dim() == 2 && clones->size(0) == 3 && counts->dim() == 1 &&
                    counts->size(0) >= 2 && clones->device() == cache_k.device() &&
                    counts->device() == cache_k.device(),
                "clones is a plan's [3, sequences], counts its [3]");
  }
  TORCH_CHECK(k.device() == cache_k.device() && v.device() == cache_k.device() &&
                  slot_map.device() == cache_k.device(),
              "all tensors must share a device");
  const c10::cuda::CUDAGuard guard(cache_k.device());
  const bc_shape s{1, int(hkv), int(hkv), int(d), 1, int(cache_k.size(0))};
  const int64_t tokens = slot_map.numel();
  check_launch(bc_append_kv(&s, int(tokens), tokens ? k.data_ptr() : nullptr, token_stride(k),
                            tokens ? v.data_ptr() : nullptr, token_stride(v), cache_k.data_ptr(),
                            cache_v.data_ptr(), &layout,
                            tokens ? slot_map.data_ptr<int>() : nullptr,
                            clones ? clones->data_ptr<int>() : nullptr,
                            clones ? int(clones->size(1)) : 0,
                            counts ? counts->data_ptr<int>() + 1 : nullptr, stream()),
               "append_kv_");
}

void run_chunk(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pages,
               const Tensor& query_start, const Tensor& lengths, Tensor& output,
               std::optional<double> scale, double softcap, int64_t window,
               const std::optional<Tensor>& alibi_slopes, const std::optional<Tensor>& prefix,
               const std::optional<Tensor>& key_start, const char* op) {
  const bc_kv_layout layout = check_cache(k, v);
  check_cuda_contiguous(pages, "pages", at::kInt);
  check_cuda_contiguous(query_start, "query_start", at::kInt);
  check_cuda_contiguous(lengths, "lengths", at::kInt);
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == k.scalar_type() && q.dim() == 3 &&
                  q.size(2) == k.size(3) && q.stride(2) == 1 &&
                  (q.size(1) == 1 || q.stride(1) == q.size(2)),
              "q must be [tokens, Hq, D] of the cache's type, each token's heads contiguous");
  const int64_t tokens = q.size(0), hq = q.size(1), hkv = k.size(2), batch = pages.size(0);
  TORCH_CHECK(hq >= 1 && hq % hkv == 0 && hq / hkv <= 128, "unsupported head counts");
  TORCH_CHECK(pages.dim() == 2 && batch >= 1 && pages.size(1) >= 1 && lengths.dim() == 1 &&
                  lengths.size(0) == batch && query_start.dim() == 1 &&
                  query_start.size(0) == batch + 1,
              "pages is [batch, max_pages], lengths [batch], query_start [batch + 1]");
  TORCH_CHECK(output.is_cuda() && output.is_contiguous() && output.sizes() == q.sizes() &&
                  (output.scalar_type() == q.scalar_type() || output.scalar_type() == at::kFloat),
              "output must be a contiguous CUDA tensor shaped like q, of q's type or FP32");
  TORCH_CHECK(tokens <= INT32_MAX && window >= 0 && window <= INT32_MAX, "window out of range");
  auto optional = [&](const std::optional<Tensor>& t, const char* name, at::ScalarType type,
                      int64_t n) -> const void* {
    if (!t) return nullptr;
    check_cuda_contiguous(*t, name, type);
    TORCH_CHECK(t->dim() == 1 && t->size(0) == n && t->device() == q.device(), name,
                " has the wrong shape or device");
    return t->data_ptr();
  };
  const bc_chunk_options options{
      float(scale ? *scale : 1.0 / std::sqrt(double(q.size(2)))), float(softcap), int(window),
      static_cast<const float*>(optional(alibi_slopes, "alibi_slopes", at::kFloat, hq)),
      static_cast<const int*>(optional(prefix, "prefix", at::kInt, batch)),
      static_cast<const int*>(optional(key_start, "key_start", at::kInt, tokens))};
  TORCH_CHECK(q.device() == k.device() && q.device() == pages.device() &&
                  q.device() == lengths.device() && q.device() == query_start.device() &&
                  q.device() == output.device(),
              "all tensors must share a device");
  if (tokens == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  const bc_shape s{int(batch), int(hq), int(hkv), int(q.size(2)), int(pages.size(1)),
                   int(k.size(0))};
  const size_t bytes = bc_chunk_workspace_bytes(&s, int(tokens));
  auto workspace = fresh({int64_t(bytes)}, at::kByte, q);
  check_launch(bc_chunk_attention(&s, int(tokens), q.scalar_type() == at::kHalf ? BC_F16 : BC_BF16,
                                  q.data_ptr(), token_stride(q), k.data_ptr(), v.data_ptr(), &layout,
                                  pages.data_ptr<int>(), query_start.data_ptr<int>(),
                                  lengths.data_ptr<int>(), &options, output.data_ptr(),
                                  output.scalar_type() == at::kFloat,
                                  bytes ? workspace.data_ptr() : nullptr, bytes, stream()),
               op);
}

Tensor chunk_attention_cuda(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& pages,
                            const Tensor& query_start, const Tensor& lengths,
                            std::optional<double> scale, double softcap, int64_t window,
                            const std::optional<Tensor>& alibi_slopes,
                            const std::optional<Tensor>& prefix,
                            const std::optional<Tensor>& key_start) {
  TORCH_CHECK(q.is_cuda(), "q must be CUDA");
  auto output = fresh(q.sizes(), q.scalar_type(), q);
  run_chunk(q, k, v, pages, query_start, lengths, output, scale, softcap, window, alibi_slopes,
            prefix, key_start, "chunk_attention");
  return output;
}

Tensor& chunk_attention_out_cuda(const Tensor& q, const Tensor& k, const Tensor& v,
                                 const Tensor& pages, const Tensor& query_start,
                                 const Tensor& lengths, Tensor& output,
                                 std::optional<double> scale, double softcap, int64_t window,
                                 const std::optional<Tensor>& alibi_slopes,
                                 const std::optional<Tensor>& prefix,
                                 const std::optional<Tensor>& key_start) {
  run_chunk(q, k, v, pages, query_start, lengths, output, scale, softcap, window, alibi_slopes,
            prefix, key_start, "chunk_attention_out");
  return output;
}

std::tuple<Tensor, Tensor, Tensor> beam_select_cuda(const Tensor& logits, const Tensor& scores,
                                                    int64_t k) {
  TORCH_CHECK(logits.is_cuda() && (is_16bit(logits) || logits.scalar_type() == at::kFloat) &&
                  logits.dim() == 3 && logits.size(0) >= 1 && logits.size(1) >= 1 &&
                  logits.size(1) <= BC_MAX_BEAMS && logits.size(2) >= 1 &&
                  logits.size(2) <= BC_MAX_BEAM_VOCAB && logits.stride(2) == 1,
              "logits must be FP16, BF16 or FP32 [batch, beams, vocab] with at most ",
              BC_MAX_BEAMS, " beams, ", BC_MAX_BEAM_VOCAB,
              " tokens and a contiguous last dimension");
  check_cuda_contiguous(scores, "scores", at::kFloat);
  const int64_t batch = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
  const int64_t row_stride = beams > 1 ? logits.stride(1) : batch > 1 ? logits.stride(0) : vocab;
  TORCH_CHECK((batch == 1 || logits.stride(0) == beams * row_stride) && row_stride >= vocab,
              "logits' rows must be equally far apart");
  TORCH_CHECK(scores.dim() == 2 && scores.size(0) == batch && scores.size(1) == beams &&
                  scores.device() == logits.device(),
              "scores must be [batch, beams] on the logits' device");
  TORCH_CHECK(k >= 1 && k <= 64 && k <= beams * vocab, "k must be in 1 .. min(64, beams * vocab)");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto out_scores = fresh({batch, k}, at::kFloat, scores);
  auto tokens = fresh({batch, k}, at::kInt, scores);
  auto parents = fresh({batch, k}, at::kInt, scores);
  const int dtype = logits.scalar_type() == at::kHalf       ? BC_F16
                    : logits.scalar_type() == at::kBFloat16 ? BC_BF16
                                                            : BC_F32;
  const size_t bytes = bc_beam_workspace_bytes(int(batch), int(beams), int(vocab), int(k), dtype);
  auto workspace = fresh({int64_t(bytes)}, at::kByte, scores);
  check_launch(bc_beam_select(int(batch), int(beams), int(vocab), int(k), dtype,
                              logits.data_ptr(), row_stride, scores.data_ptr<float>(),
                              out_scores.data_ptr<float>(), tokens.data_ptr<int>(),
                              parents.data_ptr<int>(), workspace.data_ptr(), bytes, stream()),
               "beam_select");
  return {out_scores, tokens, parents};
}

std::tuple<Tensor, Tensor> run_beam_reorder(const Tensor& pages, const Tensor& lengths,
                                            const Tensor& parents, const Tensor& refcount,
                                            const Tensor& free_stack, const Tensor& free_count,
                                            Tensor refcount_out, Tensor free_stack_out,
                                            Tensor free_count_out, const char* op) {
  const int64_t batch = pages.size(0), beams = pages.size(1), width = pages.size(2),
                out = parents.size(1);
  auto pages_out = fresh({batch, out, width}, at::kInt, pages);
  auto lengths_out = fresh({batch, out}, at::kInt, pages);
  const size_t bytes = bc_reorder_workspace_bytes(int(batch), int(beams), int(width));
  auto workspace = fresh({int64_t(bytes)}, at::kByte, pages);
  check_launch(bc_beam_reorder(int(batch), int(beams), int(out), int(refcount.numel()),
                               pages.data_ptr<int>(), int(width), lengths.data_ptr<int>(),
                               parents.data_ptr<int>(), refcount.data_ptr<int>(),
                               free_stack.data_ptr<int>(), free_count.data_ptr<int>(),
                               refcount_out.data_ptr<int>(), free_stack_out.data_ptr<int>(),
                               free_count_out.data_ptr<int>(), pages_out.data_ptr<int>(),
                               lengths_out.data_ptr<int>(), workspace.data_ptr(), bytes, stream()),
               op);
  return {pages_out, lengths_out};
}

void check_reorder(const Tensor& pages, const Tensor& lengths, const Tensor& parents,
                   const Tensor& refcount, const Tensor& free_stack, const Tensor& free_count) {
  check_state(pages, lengths, refcount, free_stack, free_count);
  check_cuda_contiguous(parents, "parents", at::kInt);
  TORCH_CHECK(pages.dim() == 3 && pages.size(0) >= 1 && pages.size(1) >= 1 &&
                  pages.size(1) <= BC_MAX_BEAMS && pages.size(2) >= 1 && lengths.dim() == 2 &&
                  lengths.size(0) == pages.size(0) && lengths.size(1) == pages.size(1) &&
                  parents.dim() == 2 && parents.size(0) == pages.size(0) &&
                  parents.size(1) >= 1 && parents.size(1) <= BC_MAX_BEAMS &&
                  parents.device() == pages.device(),
              "pages is [batch, beams, max_pages], lengths [batch, beams], parents [batch, new "
              "beams], at most ",
              BC_MAX_BEAMS, " beams, on one device");
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> beam_reorder_cuda(
    const Tensor& pages, const Tensor& lengths, const Tensor& parents, const Tensor& refcount,
    const Tensor& free_stack, const Tensor& free_count) {
  check_reorder(pages, lengths, parents, refcount, free_stack, free_count);
  const c10::cuda::CUDAGuard guard(pages.device());
  auto refcount_out = fresh(refcount.sizes(), at::kInt, pages),
       stack_out = fresh(free_stack.sizes(), at::kInt, pages),
       count_out = fresh(free_count.sizes(), at::kInt, pages);
  auto [po, lo] = run_beam_reorder(pages, lengths, parents, refcount, free_stack, free_count,
                                   refcount_out, stack_out, count_out, "beam_reorder");
  return {po, lo, refcount_out, stack_out, count_out};
}

std::tuple<Tensor, Tensor> beam_reorder_inplace_cuda(const Tensor& pages, const Tensor& lengths,
                                                     const Tensor& parents, Tensor& refcount,
                                                     Tensor& free_stack, Tensor& free_count) {
  check_reorder(pages, lengths, parents, refcount, free_stack, free_count);
  const c10::cuda::CUDAGuard guard(pages.device());
  return run_beam_reorder(pages, lengths, parents, refcount, free_stack, free_count, refcount,
                          free_stack, free_count, "beam_reorder_");
}

}  // namespace

TORCH_LIBRARY(branchcraft, m) {
  m.def("tree_verify(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor pages, Tensor lengths, "
        "Tensor draft_k, Tensor draft_v, Tensor parent) -> Tensor");
  m.def("packed_decode_out(Tensor q, Tensor packed_kv, Tensor pages, Tensor lengths, "
        "Tensor(a!) output, float scale) -> Tensor(a!)");
  m.def("commit_path_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor draft_k, Tensor draft_v, "
        "Tensor path_nodes, Tensor dest_pages, Tensor dest_slots, int request) -> ()");
  m.def("paged_decode(Tensor q, Tensor k, Tensor v, Tensor pages, Tensor lengths, "
        "int splits=0) -> Tensor");
  m.def("tree_verify_out(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor pages, "
        "Tensor lengths, Tensor draft_k, Tensor draft_v, Tensor parent, Tensor(a!) output) "
        "-> Tensor(a!)");
  m.def("packed_decode_kv_out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor pages, "
        "Tensor lengths, Tensor(a!) output, float scale, int splits=0) -> Tensor(a!)");
  m.def("commit_batch_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor draft_k, Tensor draft_v, "
        "Tensor clone_src, Tensor clone_dst, Tensor entry_request, Tensor entry_node, "
        "Tensor entry_page, Tensor entry_slot) -> ()");
  m.def("append_plan(Tensor pages, Tensor lengths, Tensor new_tokens, Tensor refcount, "
        "Tensor free_stack, Tensor free_count, int max_tokens, int max_pages=0) -> "
        "(Tensor pages, Tensor lengths, Tensor refcount, Tensor free_stack, Tensor free_count, "
        "Tensor query_start, Tensor slot_map, Tensor positions, Tensor clones, Tensor counts)");
  m.def("append_plan_(Tensor(a!) pages, Tensor(b!) lengths, Tensor new_tokens, "
        "Tensor(c!) refcount, Tensor free_stack, Tensor(d!) free_count, int max_tokens) -> "
        "(Tensor query_start, Tensor slot_map, Tensor positions, Tensor clones, Tensor counts)");
  m.def("append_kv_(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor k, Tensor v, "
        "Tensor slot_map, Tensor? clones=None, Tensor? counts=None) -> ()");
  m.def("chunk_attention(Tensor q, Tensor k, Tensor v, Tensor pages, Tensor query_start, "
        "Tensor lengths, float? scale=None, float softcap=0.0, int window=0, "
        "Tensor? alibi_slopes=None, Tensor? prefix=None, Tensor? key_start=None) -> Tensor");
  m.def("chunk_attention_out(Tensor q, Tensor k, Tensor v, Tensor pages, Tensor query_start, "
        "Tensor lengths, Tensor(a!) output, float? scale=None, float softcap=0.0, int window=0, "
        "Tensor? alibi_slopes=None, Tensor? prefix=None, Tensor? key_start=None) -> Tensor(a!)");
  m.def("beam_select(Tensor logits, Tensor scores, int k) -> (Tensor scores, Tensor tokens, "
        "Tensor parents)");
  m.def("beam_reorder(Tensor pages, Tensor lengths, Tensor parents, Tensor refcount, "
        "Tensor free_stack, Tensor free_count) -> (Tensor pages, Tensor lengths, "
        "Tensor refcount, Tensor free_stack, Tensor free_count)");
  m.def("beam_reorder_(Tensor pages, Tensor lengths, Tensor parents, Tensor(a!) refcount, "
        "Tensor(b!) free_stack, Tensor(c!) free_count) -> (Tensor pages, Tensor lengths)");
}

TORCH_LIBRARY_IMPL(branchcraft, CUDA, m) {
  m.impl("tree_verify", tree_verify_cuda);
  m.impl("packed_decode_out", packed_decode_out_cuda);
  m.impl("commit_path_", commit_path_cuda);
  m.impl("paged_decode", paged_decode_cuda);
  m.impl("tree_verify_out", tree_verify_out_cuda);
  m.impl("packed_decode_kv_out", packed_decode_kv_out_cuda);
  m.impl("commit_batch_", commit_batch_cuda);
  m.impl("append_plan", append_plan_cuda);
  m.impl("append_plan_", append_plan_inplace_cuda);
  m.impl("append_kv_", append_kv_cuda);
  m.impl("chunk_attention", chunk_attention_cuda);
  m.impl("chunk_attention_out", chunk_attention_out_cuda);
  m.impl("beam_select", beam_select_cuda);
  m.impl("beam_reorder", beam_reorder_cuda);
  m.impl("beam_reorder_", beam_reorder_inplace_cuda);
}
