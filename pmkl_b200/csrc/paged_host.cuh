// paged_host.cuh -- host side of the paged 8-bit cache's operators: argument
// checks, kernel selection and launches.  Included by pmkl_b200.cu, whose
// device checks and launch helpers it uses.
#pragma once

#include "paged_append.cuh"
#include "paged_attention_simt.cuh"
#include "paged_attention_stream.cuh"
#include "paged_attention_tile.cuh"
#include "paged_plan.cuh"

namespace pmkl_b200 {
namespace {

// SMs of the current device, asked once a device.
int cached_sm_count() {
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
        cudaGetLastError();
        return sm_count();
    }
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) known[dev].store(n = sm_count(), std::memory_order_relaxed);
    return n;
}

// Calls f with a null pointer of the element type that `dtype` names.
template <typename F>
int with_dtype(int dtype, F f) {
    if (dtype == PMKL_DTYPE_F32) return f(static_cast<float *>(nullptr));
    if (dtype == PMKL_DTYPE_F16) return f(static_cast<__half *>(nullptr));
    return f(static_cast<__nv_bfloat16 *>(nullptr));
}

unsigned blocks_for(long long units, long long per_block, int blocks_per_sm) {
    const long long need = (units + per_block - 1) / per_block;
    const long long cap = static_cast<long long>(cached_sm_count()) * blocks_per_sm;
    return static_cast<unsigned>(need < cap ? need : cap);
}

// Strides of the cache [num_blocks][kv_heads][block_size][hidden].
bool cache_view(paged::CacheView *c, const void *base, const float *scale, const int64_t *given, int kv_heads,
                int block, int hidden) {
    c->base = static_cast<uint8_t *>(const_cast<void *>(base));
    c->scale = const_cast<float *>(scale);
    const long long s[3] = {static_cast<long long>(kv_heads) * block * hidden, static_cast<long long>(block) * hidden,
                            hidden};
    for (int i = 0; i < 3; ++i) {
        if (given && given[i] < 0) return false;
        c->s[i] = given ? given[i] : s[i];
    }
    return true;
}

// (token, head) strides of a packed [tokens][heads][hidden] tensor.
bool packed_strides(long long (&st)[2], const int64_t *given, int heads, int hidden) {
    const long long s[2] = {static_cast<long long>(heads) * hidden, hidden};
    for (int i = 0; i < 2; ++i) {
        if (given && given[i] < 0) return false;
        st[i] = given ? given[i] : s[i];
    }
    return true;
}

// The tokens a request that kernel and launch are chosen for: at least one, and
// no more than there are.
int query_len(int max_query_len, int tokens) { return std::max(1, std::min(max_query_len, tokens)); }

int paged_plan_impl(const paged::PlanArgs &a, cudaStream_t stream) {
    paged::PlanArgs p = a;
    // 512 slots a CTA (1024: 8.9 us for 66 Ki tokens of 1024 requests against 6.7)
    // and at least one CTA; every CTA forms the running sums of all requests, so
    // more CTAs than SMs would only repeat them.
    const unsigned grid = p.max_tokens > 0 ? blocks_for(p.max_tokens, 512, 1) : 1;
    p.tokens_per_cta = (p.max_tokens + grid - 1) / grid;
    if (p.batch <= paged::kPlanThreads)
        paged::paged_plan_kernel<1><<<grid, paged::kPlanThreads, 0, stream>>>(p);
    else
        paged::paged_plan_kernel<4><<<grid, paged::kPlanThreads, 0, stream>>>(p);
    return launch_status();
}

template <typename T, int WPU, int NV>
int launch_append_vec(const paged::AppendArgs &p, cudaStream_t stream) {
    // Tokens a CTA: 32 (two pages of 16 rows, four runs with keys and values),
    // fewer where that would leave SMs without a CTA.
    const long long share = static_cast<long long>(p.tokens) * p.kv_heads / (4LL * cached_sm_count());
    const int span = static_cast<int>(std::min<long long>(paged::kSpanMax, std::max<long long>(2, share)));
    const long long grid = (static_cast<long long>(p.tokens) + span - 1) / span * p.kv_heads;
    if (grid > 0x7FFFFFFFLL) return PMKL_ERR_INVALID_SHAPE;
    paged::paged_append_vec_kernel<T, WPU, NV>
        <<<static_cast<unsigned>(grid), paged::kAppendThreads, 0, stream>>>(p, span);
    return launch_status();
}

// Rows of whole 16-byte vectors, at most a warp's width of them, at 16-byte
// addresses; 8-bit rows at multiples of what a lane stores.
template <typename T>
bool append_vec_applies(const paged::AppendArgs &p) {
    constexpr int kElems = 16 / sizeof(T);
    if (p.hidden % kElems != 0 || p.hidden / kElems > 32) return false;
    for (int i = 0; i < 2; ++i) {
        if (!aligned16(p.x[i]) || p.x_st[i][0] % kElems != 0 || p.x_st[i][1] % kElems != 0) return false;
        if (reinterpret_cast<uintptr_t>(p.cache[i].base) % kElems != 0) return false;
        for (long long s : p.cache[i].s)
            if (s % kElems != 0) return false;
    }
    return true;
}

int paged_append_impl(const paged::AppendArgs &p, int dtype, cudaStream_t stream) {
    return with_dtype(dtype, [&](auto *t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        if (append_vec_applies<T>(p)) {
            // A warp holds 4 KiB of a page's rows in 8 vectors a lane.
            const long long bytes = static_cast<long long>(p.block) * p.hidden * sizeof(T);
            if (bytes <= 4096) return launch_append_vec<T, 1, 8>(p, stream);
            if (bytes <= 8192) return launch_append_vec<T, 2, 8>(p, stream);
            if (bytes <= 16384) return launch_append_vec<T, 4, 8>(p, stream);
            return launch_append_vec<T, 4, 16>(p, stream);
        }
        const long long units = static_cast<long long>(p.tokens) * p.kv_heads * 2;
        paged::paged_append_kernel<T>
            <<<blocks_for(units, paged::kAppendThreads / 32, 16), paged::kAppendThreads, 0, stream>>>(p);
        return launch_status();
    });
}

// Rows of a request that share a pass over a K/V head, rounded up to the row
// tile that the stream kernel takes: 8, 16 or 32.
int stream_rows(int heads, int kv_heads, int max_q) {
    const long long rows = static_cast<long long>(heads / kv_heads) * max_q;
    return rows <= 8 ? 8 : (rows <= 16 ? 16 : 32);
}

bool stream_applies(const paged::AttnArgs &p) {
    if ((p.D != 64 && p.D != 128) || p.block % 16 != 0) return false;
    for (const paged::CacheView *c : {&p.k, &p.v}) {
        if (!aligned16(c->base)) return false;
        for (long long s : c->s)
            if (s % 16 != 0) return false;
        if (c->s[0] > 0x7FFFFFFF || c->s[2] > 0x7FFFFFFF / 16) return false;
    }
    // Rows of a request that share a K/V head, and pages' scales, are counted in 31 bits.
    return static_cast<long long>(p.tokens) * (p.H / p.Hkv) <= 0x3FFFFFFF &&
           static_cast<long long>(p.num_blocks) * p.Hkv <= 0x7FFFFFFF;
}

// Grid of a kernel that shares out `items` of at most `tiles` tiles each over
// resident CTAs (`resident`, at most `most`): no more CTAs than tiles.
long long share_grid(long long resident, long long most, long long items, long long tiles) {
    const long long grid = std::min(resident, most);
    return tiles < grid && items * tiles < grid ? std::max<long long>(1, items * tiles) : grid;
}

// Workspace addresses and alignments of the shared-out kernels.
template <typename T>
paged::StreamArgs shared_args(const paged::AttnArgs &a, void *workspace, int ctas, int rows, int tile_keys) {
    paged::StreamArgs p{};
    p.a = a;
    p.d_col = tile_keys / a.block;
    p.d_row = tile_keys % a.block;
    constexpr long long kVec = 16 / sizeof(T);
    p.vec_q = aligned16(a.q) && a.q_st[0] % kVec == 0 && a.q_st[1] % kVec == 0;
    p.vec_o = aligned16(a.o) && a.o_st[0] % kVec == 0 && a.o_st[1] % kVec == 0;
    p.k_page = static_cast<int>(a.k.s[0]);
    p.k_row = static_cast<int>(a.k.s[2]);
    p.v_page = static_cast<int>(a.v.s[0]);
    p.v_row = static_cast<int>(a.v.s[2]);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    p.desc = reinterpret_cast<paged::StreamDesc *>(ws);
    p.part_lse = reinterpret_cast<float *>(ws + ctas * sizeof(paged::StreamDesc));
    p.part_o = p.part_lse + 2LL * ctas * rows;
    return p;
}

// Launches a kernel that may be set up while the one before it in the stream
// ends; it waits on the device (griddepcontrol.wait) before it reads anything.
template <typename K>
int launch_early(K kernel, dim3 grid, int threads, int smem, const paged::StreamArgs &p, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) {
        cudaGetLastError();
        return PMKL_ERR_LAUNCH;
    }
    return PMKL_OK;
}

template <typename T, int D, int ROWS>
int launch_join(const paged::StreamArgs &p, long long grid, cudaStream_t stream) {
    // (every row that an item may have: a request may have more tokens than max_q)
    const long long rows = std::min<long long>(ROWS, static_cast<long long>(p.a.H / p.a.Hkv) * p.a.tokens);
    return launch_early(paged::paged_attention_join_kernel<T, D, ROWS>,
                        dim3(static_cast<unsigned>(grid), static_cast<unsigned>((rows + 7) / 8)),  // a warp a row
                        paged::kJoinThreads, 0, p, stream);
}

// Dynamic shared memory allowed, and CTAs an SM, asked once a device.
struct Occupancy {
    std::once_flag once[kMaxDevices];
    int per_sm[kMaxDevices] = {};
    template <typename K>
    int get(K kernel, int threads, int smem) {
        int dev = 0;
        cudaGetDevice(&dev);
        std::call_once(once[dev], [&]() {
            int n = 0;
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess &&
                cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) == cudaSuccess)
                per_sm[dev] = n;
            else
                cudaGetLastError();
        });
        return per_sm[dev];
    }
};

template <typename T, int D, int NT>
int launch_stream(const paged::AttnArgs &a, void *workspace, cudaStream_t stream) {
    using C = paged::StreamCfg<D, NT>;
    static Occupancy occupancy;
    auto kernel = paged::paged_attention_stream_kernel<T, D, NT>;
    const int per_sm = occupancy.get(kernel, C::kThreads, C::kSmemBytes);
    if (per_sm < 1) return PMKL_ERR_LAUNCH;
    const paged::StreamArgs p = shared_args<T>(a, workspace, paged::kMaxStreamCtas, C::kRows, C::kTileKeys);
    const long long tiles = std::max<long long>(
        1, (static_cast<long long>(a.max_blocks) * a.block + C::kTileKeys - 1) / C::kTileKeys);
    const long long row_tiles = (static_cast<long long>(a.H / a.Hkv) * a.max_q + C::kRows - 1) / C::kRows;
    const long long grid = share_grid(static_cast<long long>(cached_sm_count()) * per_sm, paged::kMaxStreamCtas,
                                      static_cast<long long>(a.batch) * a.Hkv * row_tiles, tiles);
    const int rc = launch_early(kernel, dim3(static_cast<unsigned>(grid)), C::kThreads, C::kSmemBytes, p, stream);
    if (rc != PMKL_OK || tiles == 1) return rc;  // an item of one tile lies in one CTA
    return launch_join<T, D, C::kRows>(p, grid, stream);
}

// The tile kernel divides its registers between its warpgroups, which needs
// the count it was written for; asked once a process.
template <typename T, int D>
bool tile_launchable() {
    static const bool ok = []() {
        cudaFuncAttributes attr;
        const bool got = cudaFuncGetAttributes(&attr, paged::paged_attention_tile_kernel<T, D>) == cudaSuccess;
        if (!got) cudaGetLastError();
        return got && attr.numRegs == paged::kTileLaunchRegs;
    }();
    return ok;
}

template <typename T, int D>
int launch_tile(const paged::AttnArgs &a, void *workspace, cudaStream_t stream) {
    using C = paged::TileCfg<D>;
    static Occupancy occupancy;
    auto kernel = paged::paged_attention_tile_kernel<T, D>;
    // Shared memory, registers and tensor memory hold two CTAs an SM (the
    // occupancy call says one of a kernel that allocates tensor memory; 296 CTAs
    // were measured to run together).
    constexpr int per_sm = 2;
    if (occupancy.get(kernel, paged::kTileThreads, C::kSmemBytes) < 1) return PMKL_ERR_LAUNCH;
    const paged::StreamArgs p = shared_args<T>(a, workspace, paged::kMaxTileCtas, paged::kTileRows, 128);
    const long long tiles = std::max<long long>(1, (static_cast<long long>(a.max_blocks) * a.block + 127) / 128);
    const long long row_tiles = (static_cast<long long>(a.H / a.Hkv) * a.max_q + 127) / 128;
    const long long grid = share_grid(static_cast<long long>(cached_sm_count()) * per_sm, paged::kMaxTileCtas,
                                      static_cast<long long>(a.batch) * a.Hkv * row_tiles, tiles);
    kernel<<<static_cast<unsigned>(grid), paged::kTileThreads, C::kSmemBytes, stream>>>(p);
    const int rc = launch_status();
    if (rc != PMKL_OK || tiles == 1) return rc;
    return launch_join<T, D, paged::kTileRows>(p, grid, stream);
}

// The tcgen05 kernel from this many rows a K/V head on (16-bit queries).  B200, 16
// requests of 500..8192 keys, 4 K/V heads of 128: 32 rows 48.8 us streaming, 53.0
// here; 40 rows (a second row tile, which reads the keys again) 73.5 and 57.1; 64
// rows 78 and 60.  One request of 131071 keys, 8 K/V heads: 32 rows 95.9 and
// 101.3, 40 rows 167 and 109; head size 64, the 16 requests: 36.3 and 38.6, 55.3
// and 42.4.
constexpr int kTileMinRows = 33;

bool many_rows(int heads, int kv_heads, int max_q) {
    return static_cast<long long>(heads / kv_heads) * max_q >= kTileMinRows;
}

int paged_attention_impl(const paged::AttnArgs &p, int dtype, int kernel, void *workspace, cudaStream_t stream) {
    const bool can_stream = stream_applies(p);
    const bool can_tile =
        can_stream && (dtype == PMKL_DTYPE_F16
                           ? (p.D == 64 ? tile_launchable<__half, 64>() : tile_launchable<__half, 128>())
                           : dtype == PMKL_DTYPE_BF16 && (p.D == 64 ? tile_launchable<__nv_bfloat16, 64>()
                                                                    : tile_launchable<__nv_bfloat16, 128>()));
    if (kernel == PMKL_PAGED_STREAM && !can_stream) return PMKL_ERR_UNSUPPORTED;
    if (kernel == PMKL_PAGED_TCGEN05 && !can_tile) return PMKL_ERR_UNSUPPORTED;
    if (can_stream && kernel != PMKL_PAGED_SIMT && p.batch > 0 && p.max_q > 0) {
        if (kernel == PMKL_PAGED_TCGEN05 || (kernel == PMKL_PAGED_AUTO && can_tile && many_rows(p.H, p.Hkv, p.max_q))) {
            if (dtype == PMKL_DTYPE_F16)
                return p.D == 64 ? launch_tile<__half, 64>(p, workspace, stream)
                                 : launch_tile<__half, 128>(p, workspace, stream);
            return p.D == 64 ? launch_tile<__nv_bfloat16, 64>(p, workspace, stream)
                             : launch_tile<__nv_bfloat16, 128>(p, workspace, stream);
        }
        const int rows = stream_rows(p.H, p.Hkv, p.max_q);
        return with_dtype(dtype, [&](auto *t) -> int {
            using T = std::remove_pointer_t<decltype(t)>;
            if (p.D == 64)
                return rows == 8    ? launch_stream<T, 64, 1>(p, workspace, stream)
                       : rows == 16 ? launch_stream<T, 64, 2>(p, workspace, stream)
                                    : launch_stream<T, 64, 4>(p, workspace, stream);
            return rows == 8    ? launch_stream<T, 128, 1>(p, workspace, stream)
                   : rows == 16 ? launch_stream<T, 128, 2>(p, workspace, stream)
                                : launch_stream<T, 128, 4>(p, workspace, stream);
        });
    }
    const long long units = static_cast<long long>(p.batch) * p.max_q * p.H;
    return with_dtype(dtype, [&](auto *t) -> int {
        using T = std::remove_pointer_t<decltype(t)>;
        paged::paged_attention_simt_kernel<T>
            <<<blocks_for(units > 0 ? units : 1, 1, 16), paged::kSimtThreads, 0, stream>>>(p);
        return launch_status();
    });
}

}  // namespace
}  // namespace pmkl_b200

extern "C" {

int pmkl_paged_plan(const int32_t *cached_lens, const int32_t *new_lens, int32_t *block_table, int64_t table_stride,
                    const int32_t *free_blocks, const int32_t *free_count, int free_capacity, int batch,
                    int max_blocks, int block_size, int64_t max_tokens, int32_t *seq_lens, int32_t *query_starts,
                    int64_t *slot_map, int32_t *free_count_out, int32_t *status, void *stream) {
    if (batch < 0 || max_blocks < 0 || block_size < 1 || max_tokens < 0 || free_capacity < 0 || table_stride < 0)
        return PMKL_ERR_INVALID_SHAPE;
    if (batch > 1 && table_stride < max_blocks) return PMKL_ERR_INVALID_SHAPE;
    if (max_tokens > 0x7FFFFFFFLL) return PMKL_ERR_INVALID_SHAPE;
    if (!free_count || !free_count_out || !query_starts) return PMKL_ERR_NULL_POINTER;
    if (free_capacity > 0 && !free_blocks) return PMKL_ERR_NULL_POINTER;
    if (max_tokens > 0 && !slot_map) return PMKL_ERR_NULL_POINTER;
    if (batch > 0 && (!cached_lens || !new_lens || !seq_lens || !status || (max_blocks > 0 && !block_table)))
        return PMKL_ERR_NULL_POINTER;
    if (free_count == free_count_out) return PMKL_ERR_INVALID_SHAPE;
    const int dev_rc = current_device_ok();
    if (dev_rc != PMKL_OK) return dev_rc;
    paged::PlanArgs p{};
    p.cached = cached_lens;
    p.fresh = new_lens;
    p.table = block_table;
    p.table_stride = table_stride;
    p.free_blocks = free_blocks;
    p.free_count = free_count;
    p.free_capacity = free_capacity;
    p.batch = batch;
    p.max_blocks = max_blocks;
    p.block = block_size;
    p.max_tokens = max_tokens;
    p.seq_lens = seq_lens;
    p.query_starts = query_starts;
    p.slots = reinterpret_cast<long long *>(slot_map);
    p.free_out = free_count_out;
    p.status = status;
    return paged_plan_impl(p, static_cast<cudaStream_t>(stream));
}

int pmkl_paged_append(const void *k, const void *v, const int64_t *k_new_strides, const int64_t *v_new_strides,
                      const int64_t *slot_map, int tokens, int kv_heads, int hidden, int dtype, void *k_cache,
                      void *v_cache, const int64_t *k_strides, const int64_t *v_strides, float *k_scale,
                      float *v_scale, int num_blocks, int block_size, void *stream) {
    if (tokens < 0 || kv_heads < 0 || hidden < 0 || num_blocks < 0 || block_size < 1) return PMKL_ERR_INVALID_SHAPE;
    if (!dtype_valid(dtype)) return PMKL_ERR_INVALID_DTYPE;
    if (tokens == 0 || kv_heads == 0 || hidden == 0 || num_blocks == 0) return PMKL_OK;
    if (hidden > 256) return PMKL_ERR_UNSUPPORTED;
    if (!k || !v || !slot_map || !k_cache || !v_cache || !k_scale || !v_scale) return PMKL_ERR_NULL_POINTER;
    paged::AppendArgs p{};
    p.x[0] = k;
    p.x[1] = v;
    if (!packed_strides(p.x_st[0], k_new_strides, kv_heads, hidden) ||
        !packed_strides(p.x_st[1], v_new_strides, kv_heads, hidden) ||
        !cache_view(&p.cache[0], k_cache, k_scale, k_strides, kv_heads, block_size, hidden) ||
        !cache_view(&p.cache[1], v_cache, v_scale, v_strides, kv_heads, block_size, hidden))
        return PMKL_ERR_INVALID_SHAPE;
    const int dev_rc = current_device_ok();
    if (dev_rc != PMKL_OK) return dev_rc;
    p.slots = reinterpret_cast<const long long *>(slot_map);
    p.tokens = tokens;
    p.kv_heads = kv_heads;
    p.hidden = hidden;
    p.block = block_size;
    p.num_slots = static_cast<long long>(num_blocks) * block_size;
    return paged_append_impl(p, dtype, static_cast<cudaStream_t>(stream));
}

size_t pmkl_paged_attention_workspace_size_ex(int tokens, int batch, int heads, int kv_heads, int hidden,
                                              int max_query_len, int dtype, int kernel) {
    if (tokens <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || hidden <= 0 || max_query_len < 0 ||
        heads % kv_heads != 0 || !dtype_valid(dtype))
        return 0;
    max_query_len = query_len(max_query_len, tokens);
    // The CUDA-core kernel needs none.
    if ((hidden != 64 && hidden != 128) || kernel == PMKL_PAGED_SIMT) return 0;
    size_t need = 0;
    // (the streaming kernel also where the tcgen05 kernel is chosen and does not fit)
    if (kernel != PMKL_PAGED_TCGEN05)
        need = paged::partial_workspace(paged::kMaxStreamCtas, stream_rows(heads, kv_heads, max_query_len), hidden);
    if (dtype != PMKL_DTYPE_F32 && (kernel == PMKL_PAGED_TCGEN05 || (kernel == PMKL_PAGED_AUTO && many_rows(heads, kv_heads, max_query_len))))
        need = std::max(need, paged::partial_workspace(paged::kMaxTileCtas, paged::kTileRows, hidden));
    return align256(need);
}

size_t pmkl_paged_attention_workspace_size(int tokens, int batch, int heads, int kv_heads, int hidden,
                                           int max_query_len, int dtype) {
    size_t need = 0;
    for (int kernel : {PMKL_PAGED_STREAM, PMKL_PAGED_TCGEN05})
        need = std::max(need, pmkl_paged_attention_workspace_size_ex(tokens, batch, heads, kv_heads, hidden,
                                                                     max_query_len, dtype, kernel));
    return need;
}

int pmkl_paged_attention(const void *q, const int64_t *q_strides, const void *k_cache, const void *v_cache,
                         const int64_t *k_strides, const int64_t *v_strides, const float *k_scale,
                         const float *v_scale, const int32_t *block_table, int64_t table_stride,
                         const int32_t *seq_lens, const int32_t *query_starts, void *o, const int64_t *o_strides,
                         float *lse, int tokens, int batch, int heads, int kv_heads, int hidden, int num_blocks,
                         int block_size, int max_blocks, int max_query_len, int dtype, int is_causal, float scale,
                         void *workspace, size_t workspace_bytes, int kernel, void *stream) {
    if (tokens < 0 || batch < 0 || heads < 0 || kv_heads < 0 || hidden < 0 || num_blocks < 0 || block_size < 1 ||
        max_blocks < 0 || max_query_len < 0 || table_stride < 0)
        return PMKL_ERR_INVALID_SHAPE;
    if (!dtype_valid(dtype)) return PMKL_ERR_INVALID_DTYPE;
    if (kernel != PMKL_PAGED_AUTO && kernel != PMKL_PAGED_SIMT && kernel != PMKL_PAGED_STREAM &&
        kernel != PMKL_PAGED_TCGEN05) return PMKL_ERR_UNSUPPORTED;
    if (heads > 0 && (kv_heads == 0 || heads % kv_heads != 0)) return PMKL_ERR_INVALID_SHAPE;
    if (batch > 1 && table_stride < max_blocks) return PMKL_ERR_INVALID_SHAPE;
    if (!query_starts && tokens != batch) return PMKL_ERR_INVALID_SHAPE;
    if (!query_starts) max_query_len = 1;
    if (heads > 0 && static_cast<long long>(max_query_len) * (heads / kv_heads) > 0x3FFFFFFFLL)
        return PMKL_ERR_INVALID_SHAPE;
    if (tokens == 0 || heads == 0 || hidden == 0) return PMKL_OK;
    if (hidden > 256) return PMKL_ERR_UNSUPPORTED;
    if (!q || !o) return PMKL_ERR_NULL_POINTER;
    if (batch > 0 && !seq_lens) return PMKL_ERR_NULL_POINTER;
    if (batch > 0 && max_blocks > 0 && !block_table) return PMKL_ERR_NULL_POINTER;
    if (num_blocks > 0 && (!k_cache || !v_cache || !k_scale || !v_scale)) return PMKL_ERR_NULL_POINTER;
    const size_t need =
        pmkl_paged_attention_workspace_size_ex(tokens, batch, heads, kv_heads, hidden, max_query_len, dtype, kernel);
    if (need > 0) {
        if (!workspace) return PMKL_ERR_NULL_POINTER;
        if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return PMKL_ERR_MISALIGNED;
        if (workspace_bytes < need) return PMKL_ERR_WORKSPACE;
    }
    paged::AttnArgs p{};
    if (!packed_strides(p.q_st, q_strides, heads, hidden) || !packed_strides(p.o_st, o_strides, heads, hidden) ||
        !cache_view(&p.k, k_cache, k_scale, k_strides, kv_heads, block_size, hidden) ||
        !cache_view(&p.v, v_cache, v_scale, v_strides, kv_heads, block_size, hidden))
        return PMKL_ERR_INVALID_SHAPE;
    const int dev_rc = current_device_ok();
    if (dev_rc != PMKL_OK) return dev_rc;
    p.q = q;
    p.o = o;
    p.table = block_table;
    p.table_stride = table_stride;
    p.seq_lens = seq_lens;
    p.query_starts = query_starts;
    p.lse = lse;
    p.tokens = tokens;
    p.batch = batch;
    p.H = heads;
    p.Hkv = kv_heads;
    p.D = hidden;
    p.num_blocks = num_blocks;
    p.block = block_size;
    p.max_blocks = max_blocks;
    p.max_q = query_len(max_query_len, tokens);
    p.causal = is_causal ? 1 : 0;
    // (below the normal numbers a score scale is as good as the smallest of them)
    p.scale = scale > 0.f ? fmaxf(scale, 1.17549435e-38f) : 1.0f / sqrtf(static_cast<float>(hidden));
    return paged_attention_impl(p, dtype, kernel, workspace, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
