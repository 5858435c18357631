// The paged 8-bit cache's operators for torch: checks of the tensors, outputs
// and workspace from torch's allocator, the C ABI on the current stream.
// Included by fused_self_attention.cpp.  No reference counterpart.
#pragma once

#include <ATen/cuda/EmptyTensor.h>

namespace {

// At the small end these calls are bound by what the host does: outputs come
// straight from the allocator, and several from one allocation.
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType type, const at::Device &dev) {
    return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

// Elements [from, from + n) of a contiguous vector, sharing its memory.
at::Tensor part_of(const at::Tensor &base, int64_t from, int64_t n) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(base.storage()),
                                                     base.key_set(), base.dtype());
    impl->set_storage_offset(from);
    impl->set_sizes_contiguous({n});
    return at::Tensor(std::move(impl));
}

void check_i32(const at::Tensor &t, const char *name, int64_t dims, const at::Device &dev) {
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dims, name, " must be an int32 tensor of ", dims,
                " dimension(s)");
    TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
}

void check_vector(const at::Tensor &t, const char *name, int64_t n, const at::Device &dev) {
    check_i32(t, name, 1, dev);
    TORCH_CHECK(t.numel() == n && (n <= 1 || t.stride(0) == 1), name, " must be contiguous, of ", n, " elements");
}

// A cache tensor [pages, kv_heads, block, hidden] and its scales [pages, kv_heads].
void check_cache(const at::Tensor &c, const at::Tensor &s, const char *name, const at::Device &dev) {
    TORCH_CHECK(c.dim() == 4 && (c.scalar_type() == at::ScalarType::Float8_e4m3fn || c.scalar_type() == at::kByte),
                name, "_cache must be a float8_e4m3fn (or uint8) tensor [pages, kv_heads, block, hidden]");
    TORCH_CHECK(c.device() == dev && s.device() == dev, name, "_cache and ", name, "_scale must be on ", dev);
    TORCH_CHECK(c.size(3) <= 1 || c.stride(3) == 1, name, "_cache must be contiguous in its hidden dimension");
    TORCH_CHECK(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == c.size(0) && s.size(1) == c.size(1) &&
                    s.is_contiguous(),
                name, "_scale must be a contiguous float32 tensor [pages, kv_heads]");
    for (int i = 0; i < 4; ++i) TORCH_CHECK(c.size(i) <= INT32_MAX, name, "_cache: sizes must fit in 32-bit integers");
}

std::array<int64_t, 3> cache_strides(const at::Tensor &c) { return {c.stride(0), c.stride(1), c.stride(2)}; }

void check_packed(const at::Tensor &t, const char *name) {
    TORCH_CHECK(t.is_cuda(), name, ": the paged operators run on CUDA tensors only; got a CPU tensor");
    TORCH_CHECK(t.dim() == 3 && pmkl_dtype_of(t.scalar_type()) >= 0, name,
                " must be a float32, float16 or bfloat16 tensor [tokens, heads, hidden]");
    for (int i = 0; i < 3; ++i) TORCH_CHECK(t.size(i) <= INT32_MAX, name, ": sizes must fit in 32-bit integers");
}

at::Tensor packed_rows(const at::Tensor &t) { return t.size(2) <= 1 || t.stride(2) == 1 ? t : t.contiguous(); }

void check_table(const at::Tensor &t, int64_t batch, const at::Device &dev) {
    check_i32(t, "block_table", 2, dev);
    TORCH_CHECK(t.size(0) == batch && (t.size(1) <= 1 || t.stride(1) == 1) && t.size(1) <= INT32_MAX,
                "block_table must be [batch, pages], its rows contiguous");
    TORCH_CHECK(batch <= 1 || t.stride(0) >= t.size(1), "block_table: rows must not overlap");
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> paged_plan(
    const at::Tensor &cached_lens, const at::Tensor &new_lens, const at::Tensor &block_table,
    const at::Tensor &free_blocks, const at::Tensor &free_count, int64_t block_size, int64_t max_tokens) {
    TORCH_CHECK(cached_lens.is_cuda(), "paged_plan runs on CUDA tensors only; got a CPU tensor");
    const at::Device dev = cached_lens.device();
    const int64_t batch = cached_lens.dim() == 1 ? cached_lens.size(0) : 0;
    TORCH_CHECK(batch <= INT32_MAX - 1, "paged_plan: batch must fit in a 32-bit integer");
    check_vector(cached_lens, "cached_lens", batch, dev);
    check_vector(new_lens, "new_lens", batch, dev);
    check_table(block_table, batch, dev);
    check_i32(free_blocks, "free_blocks", 1, dev);
    check_vector(free_blocks, "free_blocks", free_blocks.numel(), dev);
    TORCH_CHECK(free_blocks.numel() <= INT32_MAX, "paged_plan: free_blocks has too many elements");
    check_vector(free_count, "free_count", 1, dev);
    TORCH_CHECK(block_size >= 1 && block_size <= INT32_MAX && max_tokens >= 0 && max_tokens <= INT32_MAX,
                "paged_plan: block_size must be positive and max_tokens not negative");
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor ints = new_tensor({3 * batch + 2}, at::kInt, dev);
    at::Tensor slot_map = new_tensor({max_tokens}, at::kLong, dev);
    at::Tensor seq_lens = part_of(ints, 0, batch), status = part_of(ints, batch, batch);
    at::Tensor starts = part_of(ints, 2 * batch, batch + 1), left = part_of(ints, 3 * batch + 1, 1);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const int rc = pmkl_paged_plan(
        cached_lens.data_ptr<int>(), new_lens.data_ptr<int>(), block_table.data_ptr<int>(),
        batch > 1 ? block_table.stride(0) : block_table.size(1), free_blocks.data_ptr<int>(),
        free_count.data_ptr<int>(), static_cast<int>(free_blocks.numel()), static_cast<int>(batch),
        static_cast<int>(block_table.size(1)), static_cast<int>(block_size), max_tokens, seq_lens.data_ptr<int>(),
        starts.data_ptr<int>(), slot_map.data_ptr<int64_t>(), left.data_ptr<int>(), status.data_ptr<int>(), stream);
    TORCH_CHECK(rc == PMKL_OK, "pmkl_paged_plan failed: ", pmkl_status_string(rc));
    return std::make_tuple(seq_lens, starts, slot_map, left, status);
}

void paged_append(const at::Tensor &k, const at::Tensor &v, const at::Tensor &slot_map, const at::Tensor &k_cache,
                  const at::Tensor &v_cache, const at::Tensor &k_scale, const at::Tensor &v_scale) {
    check_packed(k, "k");
    check_packed(v, "v");
    const at::Device dev = k.device();
    TORCH_CHECK(k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && v.device() == dev,
                "paged_append: k and v must have the same shape, dtype and device");
    check_cache(k_cache, k_scale, "k", dev);
    check_cache(v_cache, v_scale, "v", dev);
    TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "paged_append: k_cache and v_cache must have the same shape");
    TORCH_CHECK(k.size(1) == k_cache.size(1) && k.size(2) == k_cache.size(3),
                "paged_append: k and v must have the cache's heads and hidden size");
    TORCH_CHECK(slot_map.scalar_type() == at::kLong && slot_map.dim() == 1 && slot_map.size(0) == k.size(0) &&
                    slot_map.is_contiguous() && slot_map.device() == dev,
                "paged_append: slot_map must be a contiguous int64 tensor of a slot for each token");
    TORCH_CHECK(k_cache.size(2) >= 1, "paged_append: pages must have rows");
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor kc = packed_rows(k), vc = packed_rows(v);
    const int64_t ks[2] = {kc.stride(0), kc.stride(1)}, vs[2] = {vc.stride(0), vc.stride(1)};
    const auto kst = cache_strides(k_cache), vst = cache_strides(v_cache);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const int rc = pmkl_paged_append(
        kc.data_ptr(), vc.data_ptr(), ks, vs, slot_map.data_ptr<int64_t>(), static_cast<int>(k.size(0)),
        static_cast<int>(k.size(1)), static_cast<int>(k.size(2)), pmkl_dtype_of(k.scalar_type()), k_cache.data_ptr(),
        v_cache.data_ptr(), kst.data(), vst.data(), k_scale.data_ptr<float>(), v_scale.data_ptr<float>(),
        static_cast<int>(k_cache.size(0)), static_cast<int>(k_cache.size(2)), stream);
    TORCH_CHECK(rc == PMKL_OK, "pmkl_paged_append failed: ", pmkl_status_string(rc));
}

std::tuple<at::Tensor, at::Tensor> paged_attention_fw(
    const at::Tensor &q, const at::Tensor &k_cache, const at::Tensor &v_cache, const at::Tensor &k_scale,
    const at::Tensor &v_scale, const at::Tensor &block_table, const at::Tensor &seq_lens,
    const c10::optional<at::Tensor> &query_starts, c10::optional<int64_t> max_len, bool is_causal, double scale,
    int64_t kernel) {
    check_packed(q, "q");
    const at::Device dev = q.device();
    check_cache(k_cache, k_scale, "k", dev);
    check_cache(v_cache, v_scale, "v", dev);
    TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "paged_attention: k_cache and v_cache must have the same shape");
    TORCH_CHECK(q.size(2) == k_cache.size(3) && k_cache.size(1) > 0 && q.size(1) % k_cache.size(1) == 0,
                "paged_attention: the cache must have q's hidden size and heads dividing q's heads");
    const int64_t batch = seq_lens.dim() == 1 ? seq_lens.size(0) : 0;
    TORCH_CHECK(batch <= INT32_MAX - 1, "paged_attention: batch must fit in a 32-bit integer");
    check_vector(seq_lens, "seq_lens", batch, dev);
    check_table(block_table, batch, dev);
    if (query_starts.has_value())
        check_vector(*query_starts, "query_starts", batch + 1, dev);
    else
        TORCH_CHECK(q.size(0) == batch, "paged_attention: without query_starts q must have one token a request");
    // Not given: the requests' average, since it only chooses the kernel.
    const int64_t max_query_len = max_len.has_value() ? *max_len : (q.size(0) + batch - 1) / std::max<int64_t>(batch, 1);
    TORCH_CHECK(max_query_len >= 0 && max_query_len <= INT32_MAX, "paged_attention: max_query_len must not be negative");
    TORCH_CHECK(k_cache.size(2) >= 1, "paged_attention: pages must have rows");
    const c10::cuda::CUDAGuard guard(dev);
    const at::Tensor qc = packed_rows(q);
    const int64_t qs[2] = {qc.stride(0), qc.stride(1)};
    const auto kst = cache_strides(k_cache), vst = cache_strides(v_cache);
    const int T = static_cast<int>(q.size(0)), H = static_cast<int>(q.size(1)), D = static_cast<int>(q.size(2));
    const int Hkv = static_cast<int>(k_cache.size(1)), dt = pmkl_dtype_of(q.scalar_type());
    at::Tensor out = new_tensor(q.sizes(), q.scalar_type(), dev);
    at::Tensor lse = new_tensor({q.size(0), q.size(1)}, at::kFloat, dev);
    const size_t ws_bytes = pmkl_paged_attention_workspace_size_ex(
        T, static_cast<int>(batch), H, Hkv, D, static_cast<int>(max_query_len), dt, static_cast<int>(kernel));
    at::Tensor ws;
    if (ws_bytes > 0) ws = new_tensor({static_cast<int64_t>(ws_bytes)}, at::kByte, dev);
    cudaStream_t stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const int rc = pmkl_paged_attention(
        qc.data_ptr(), qs, k_cache.data_ptr(), v_cache.data_ptr(), kst.data(), vst.data(), k_scale.data_ptr<float>(),
        v_scale.data_ptr<float>(), block_table.data_ptr<int>(),
        batch > 1 ? block_table.stride(0) : block_table.size(1), seq_lens.data_ptr<int>(),
        query_starts.has_value() ? query_starts->data_ptr<int>() : nullptr, out.data_ptr(), nullptr,
        lse.data_ptr<float>(), T, static_cast<int>(batch), H, Hkv, D, static_cast<int>(k_cache.size(0)),
        static_cast<int>(k_cache.size(2)), static_cast<int>(block_table.size(1)), static_cast<int>(max_query_len), dt,
        is_causal ? 1 : 0, static_cast<float>(scale), ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
        static_cast<int>(kernel), stream);
    TORCH_CHECK(rc == PMKL_OK, "pmkl_paged_attention failed: ", pmkl_status_string(rc));
    return std::make_tuple(out, lse);
}
