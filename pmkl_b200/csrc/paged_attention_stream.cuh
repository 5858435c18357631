// paged_attention_stream.cuh -- attention of a few query rows a request over
// the paged 8-bit cache: head size 64 or 128, pages of a multiple of 16 rows.
//
// The rows of a request that read one K/V head (its tokens times the query
// heads of the group) share one pass over that head's cache, 2 D bytes a key
// for 4 D FLOP a row: with up to a few tens of rows the cache's bytes are the
// bound, so the kernel is built to keep loads in flight and nothing else.
//
//   * Work is the list of all (request, K/V head, row tile) items, each cut in
//     tiles of 16 keys a warp (128 keys; 192 with 9 to 16 rows); a grid of resident CTAs takes equal shares of the
//     list, whatever the lengths, a CTA's share beginning and ending inside an
//     item.  Each CTA finds its share from the lengths itself.  Items that lie
//     in one CTA are written at once; the others leave normalised partial rows
//     and their log-sums in the workspace, joined in the list's order by a
//     second kernel (no atomics: the same bits on every run).  Two or more
//     shares a resident CTA balance no better than they cost (B200, 16 x 4096
//     keys, 32 heads: 99 us with one, 104 with two, 111 with three).
//   * A warp takes 16 keys at a time, copied asynchronously to shared memory of
//     its own two tiles ahead (4 KB a tile at head size 128, 64 KB an SM under
//     way), and reads them as the operands of the tensor cores: a sum over D may
//     run in any order, so thread (g, t) = (lane / 4, lane % 4) takes 16
//     consecutive bytes of keys g and g + 8 and the queries are laid out to
//     match; and output rows may come in any order, so for V it takes 16
//     consecutive bytes of keys 2t, 2t + 1, 2t + 8, 2t + 9 and pairs up the
//     bytes of neighbouring keys.  e4m3 values are exact in fp16, which is what
//     the products take.  (Loads into registers instead ran as fast where the
//     compiler kept them apart and up to 18 % slower where it did not.)
//   * S^T = K Q^T puts keys in rows and queries in columns; its result is
//     turned into the operand of O^T = V^T P^T by a transposing matrix move.
//   * 16-bit queries go to fp16 over a power of two that brings the row's largest
//     value near 2^7: exact but for what lies below 2^-32 of it.  fp32 queries
//     and weights are split in two fp16 parts (2^-22 of themselves).
//   * A page's value scale enters the exponent: w = s + log2 vs, p' = 2^(w - M)
//     rounded to fp16 for the product, and the sum of the softmax takes p' / vs
//     in fp32.  M is such that weights go up to 2^15, so that small ones keep what
//     fp16 has below: it is raised only when some w would pass that, to where the
//     largest is 2^7 (voted per warp), so most tiles reduce nothing across lanes.
//     What a weight may lose beside 2^-11 of itself is then 2^-32 of the largest.
//     fp32 queries raise M to where the largest weight is 2^13: 2^-22 of a weight
//     or 2^-38 of the largest.  Where vs is small and another page's large, p' may
//     be 0 and p' / vs not: pages of small vs add 2^(w - M - log2 vs) to the sum.
//
// mma.sync and not tcgen05: 8 to 32 query rows leave most of a 128-row tcgen05
// tile empty, and the cache's bytes are the bound.  B200, device time: 16 x 4096
// keys, 32 heads of 128 (538 MB): 102 us, 5.27 TB/s (0.80 of the measured copy
// bandwidth; a CTA's loop over tiles alone runs at 7.6 TB/s, the rest is its
// start of some 8000 cycles, the change of items and the join); 64 requests of
// 1..16384 keys, 32/8 heads (939 MB): 188 us, 5.0 TB/s; one request of 131071
// keys, 32/8 heads (269 MB): 62 us; 8 x 1024 keys, 16 heads of 64: 14.0 us and
// 2 x 128 keys, 4 heads, fp32: 6.4 us, bound by the latency of what comes before
// the first key (lengths, share, table, queries) and of the join.
//
// Rows behind a request's last key may hold anything: their scores are set to
// -inf by selection and their values to zero.  A key that some rows see and
// others do not (a later token of the same step) may hold NaN too, which the
// product would spread as 0 * NaN: tiles at the diagonal look for NaN bytes,
// and where there are any the product gets zeros for them and the rows that do
// see the key note its columns.
#pragma once

#include "paged_attention_simt.cuh"

namespace pmkl_b200 {
namespace paged {

constexpr int kMaxStreamCtas = 640;           // partials in the workspace: 148 SMs with up to 4 CTAs

// Workspace: an item descriptor a CTA, then log-sums [2 CTAs][rows], then
// partial rows [2 CTAs][rows][D].  A CTA's slot 2c holds the item that it
// enters in the middle, 2c + 1 the item that it begins and does not end.
struct StreamDesc {
    int segments;  // CTAs that the item is spread over; 0: none
    int first, h, row0, n_rows;
    int pad[3];
};

struct StreamArgs {
    AttnArgs a;
    int vec_q, vec_o;  // rows of q, of o are 16-byte aligned
    int d_col, d_row;  // keys of a tile as pages and rows of one
    int k_page, k_row, v_page, v_row;  // bytes from page to page and row to row of the cache, where 31 bits hold them
    float *part_o, *part_lse;
    StreamDesc *desc;
};

__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint32_t v) {  // the low 16 bits
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_h2_hi(uint32_t v) {  // the high 16 bits
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(v));
    return r;
}

// c += a b, a 16 x 16 (rows g, g + 8), b 16 x 8 fp16, c 16 x 8 fp32.
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ uint32_t h2_bits(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 h2_floats(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }

// A running maximum before its first score: no fp32 number is below it, and it is
// finite, so that differences with it are numbers.
constexpr float kNoMax = -3.402823466e38f;

// Weights are 2^(w - M) up to 2^kTopExp, where fp16 ends; M is raised to where the
// largest is 2^lift.
constexpr float kTopExp = 15.f;
template <typename T>
constexpr float kLift = sizeof(T) == 4 ? 13.f : 7.f;

// log2 of the value scales below which the sum's terms come from exponents of their
// own.  From there on, 2^(7 - 32 - 64) in front of a weight, one of 2^-37 of the
// largest is still a normal number, whatever the scale of the other pages.
constexpr float kSmallScale = -32.f;

__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The square root of 2^x: sums as large as 1 / vs are multiplied by it twice where
// 2^x itself would be 0 (x down to -252).
__device__ __forceinline__ float exp2_half(float x) { return exp2_fast(0.5f * x); }

// Asynchronous copies to shared memory: 16 bytes past L1 (a step reads the cache
// once), or 4.
__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }
__device__ __forceinline__ uint4 shared16(uint32_t at) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at) : "memory");
    return r;
}
__device__ __forceinline__ uint2 shared8(uint32_t at) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at) : "memory");
    return r;
}

// 16 bytes, or zeros where `there` is false: predicated, not branched around.
__device__ __forceinline__ uint4 load16_if(const uint8_t *p, bool there) {
    uint4 r = make_uint4(0, 0, 0, 0);
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
        "@p ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
        : "l"(p), "r"(there ? 1u : 0u));
    return r;
}

template <int D, int NT>
struct StreamCfg {
    static constexpr int kRows = 8 * NT;
    // Two CTAs of 8 warps an SM where 128 registers a thread do; one of 12 or 8
    // where the accumulators of 16 or 32 rows need more.
    static constexpr int kWarps = NT == 2 ? 12 : 8;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kTileKeys = 16 * kWarps;  // keys a CTA takes at a time
    static constexpr int kItemCost = 3;            // of an item, in tiles: some 8000 cycles against 2450 (16 x 4096 keys)
    static constexpr int kRowPitch = D + 32;  // 4 floats behind every D / 8: a warp's float4 stores meet no bank twice
    // Two stages of 16 keys and values a warp, and their scales.
    static constexpr int kStageBytes = 2 * 16 * D + 16;
    static constexpr int kDataBytes = kWarps * 2 * kStageBytes;
    // The warps' sums: one warp each, or (16 and 32 rows) two adding to one.
    static constexpr int kSlots = NT == 1 ? kWarps : kWarps / 2;
    static constexpr int kAccBytes = kSlots * kRows * kRowPitch * 4;
    // The query operands, 8 bytes a lane and step, for two fp16 parts.
    static constexpr int kSmemBytes = kDataBytes + kAccBytes + 2 * NT * (D / 16) * 32 * 8;
};

__host__ __device__ constexpr size_t partial_workspace(int ctas, int rows, int D) {
    return static_cast<size_t>(ctas) * (sizeof(StreamDesc) + 2 * static_cast<size_t>(rows) * (D + 1) * 4);
}

// The work of both kernels that share it out: items are (request, K/V head,
// ROWS rows), in that order, each cut in tiles of KEYS keys up to the last key
// that its rows see, at least one, so that every item has a writer.  The list
// counts an item as its tiles and COST more, the tiles' worth of what a CTA
// does once for an item (queries, first loads, join, output): shares of many
// short items then take no longer than shares of one long.  The COST comes
// first: a share that begins or ends in it begins or ends at tile 0.

// One stretch of an item's key tiles.
struct Segment {
    Request r;
    int b, h, row0, n_rows, tile0, tile1, tiles;
    int lim_min, lim_max;  // keys that the first and last row see
    int last_cta;          // where the item ends in a later CTA: which
};

// The share of a CTA in the list of tiles, and the walk through it.
struct Share {
    long long total, shares, u, u_end, b_begin;
    int b;
    // The stretch that comes next, once `placed`: request, head, first row, the
    // place in the item (COST counted) and its tiles.
    bool placed;
    Request r;
    int h, row0, at, tiles;
};

// Where share c of `shares` begins in `total` tiles (and, with the two exchanged,
// near which share a tile lies).  32-bit division where it does: the 64-bit one is
// a long routine.
__host__ __device__ __forceinline__ long long share_begin(long long total, long long c, long long shares) {
    const unsigned long long n = static_cast<unsigned long long>(total) * c;
    return ((n | shares) >> 32) == 0 ? static_cast<unsigned>(n) / static_cast<unsigned>(shares) : n / shares;
}
__host__ __device__ __forceinline__ int quotient(long long a, long long b) {  // a, b >= 0, the result an int
    return ((a | b) >> 32) == 0 ? static_cast<unsigned>(a) / static_cast<unsigned>(b) : static_cast<int>(a / b);
}

template <int ROWS, int KEYS, int COST>
__host__ __device__ __forceinline__ int tile_count(const AttnArgs &p, const Request &r, int row0, int rows, int group) {
    return max(1, (visible(p, r, (min(row0 + ROWS, rows) - 1) / group) + KEYS - 1) / KEYS);
}

// What the row tiles of a request come to, for one K/V head.
template <int ROWS, int KEYS, int COST>
__host__ __device__ __forceinline__ long long head_tiles(const AttnArgs &p, const Request &r, int group) {
    const int rows = r.rows * group;
    long long n = 0;
#pragma unroll 1
    for (int row0 = 0; row0 < rows; row0 += ROWS) n += COST + tile_count<ROWS, KEYS, COST>(p, r, row0, rows, group);
    return n;
}

template <int ROWS, int KEYS, int COST>
__device__ __noinline__ long long request_weight(const AttnArgs &p, int b) {
    return head_tiles<ROWS, KEYS, COST>(p, request_of(p, b), p.H / p.Hkv) * p.Hkv;
}

// The next stretch of one item in the share.  The first is found by division;
// from there the walk steps from row tile to row tile, head to head, request to
// request.
template <int ROWS, int KEYS, int COST>
__host__ __device__ __forceinline__ bool next_segment(const AttnArgs &p, Share &w, Segment &s) {
    const int group = p.H / p.Hkv;
    if (w.u >= w.u_end) return false;
    if (!w.placed) {
        w.placed = true;
        w.r = request_of(p, w.b);
        const long long per_head = head_tiles<ROWS, KEYS, COST>(p, w.r, group);
        w.h = quotient(w.u - w.b_begin, per_head);
        long long left = (w.u - w.b_begin) - w.h * per_head;
        w.row0 = 0;
        w.tiles = tile_count<ROWS, KEYS, COST>(p, w.r, 0, w.r.rows * group, group);
#pragma unroll 1
        while (left >= w.tiles + COST) {
            left -= w.tiles + COST;
            w.row0 += ROWS;
            w.tiles = tile_count<ROWS, KEYS, COST>(p, w.r, w.row0, w.r.rows * group, group);
        }
        w.at = static_cast<int>(left);
    }
    // The share's part of the item: from `at` (COST counted) as far as the share goes.
    if (w.u_end - w.u <= COST - w.at) return false;  // no tile of it
    const int rows = w.r.rows * group;
    const int end = static_cast<int>(min(static_cast<long long>(w.tiles) + COST, w.at + (w.u_end - w.u)));
    s.r = w.r;
    s.b = w.b;
    s.h = w.h;
    s.row0 = w.row0;
    s.n_rows = min(ROWS, rows - w.row0);
    s.tiles = w.tiles;
    s.tile0 = max(0, w.at - COST);
    s.tile1 = end - COST;
    s.lim_min = visible(p, w.r, w.row0 / group);
    s.lim_max = visible(p, w.r, (w.row0 + s.n_rows - 1) / group);
    w.u += end - w.at;
    if (s.tile1 < s.tiles) {
        // The CTA whose share holds the item's last tile; this is the share's last stretch.
        const long long last = w.u + (s.tiles - s.tile1) - 1;
        long long c = share_begin(w.shares, last, w.total);  // within one of the owner
        while (share_begin(w.total, c + 1, w.shares) <= last) ++c;
        while (share_begin(w.total, c, w.shares) > last) --c;
        s.last_cta = static_cast<int>(c);
    } else if (w.u < w.u_end) {
        w.at = 0;
        w.row0 += ROWS;
        if (w.row0 >= rows) {
            w.row0 = 0;
            if (++w.h == p.Hkv) {
                w.h = 0;
                do {
                    if (++w.b >= p.batch) {  // (lengths that changed under the kernel)
                        w.u_end = w.u;
                        return true;
                    }
                    w.r = request_of(p, w.b);
                } while (w.r.rows == 0);
            }
        }
        w.tiles = tile_count<ROWS, KEYS, COST>(p, w.r, w.row0, w.r.rows * group, group);
    }
    return true;
}

// Finds the CTA's share: called by all THREADS threads, `sum` one value a warp,
// the result in `to` (visible after the next __syncthreads).
template <int ROWS, int KEYS, int COST, int THREADS>
__device__ __forceinline__ void find_share(const AttnArgs &p, long long (&sum)[THREADS / 32], Share &to) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const auto weight = [&](int b) -> long long { return b < p.batch ? request_weight<ROWS, KEYS, COST>(p, b) : 0; };
    // Inclusive sum over the block; `sum` then holds the warps' own.
    const auto inclusive = [&](long long v) -> long long {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += x;
        }
        __syncthreads();
        if (lane == 31) sum[warp] = v;
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < warp; ++w) v += sum[w];
        return v;
    };
    const bool one = p.batch <= THREADS;  // a request a thread: one sum does
    long long part = 0, total = 0;
#pragma unroll 1
    for (int b = tid; b < p.batch; b += THREADS) part += weight(b);
    const long long upto = inclusive(part);
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) total += sum[w];
    // As many shares as CTAs, or as tiles where those are fewer: none is empty.
    const long long shares = min(total, static_cast<long long>(gridDim.x));
    const bool idle = blockIdx.x >= shares;
    const long long u = idle ? 0 : share_begin(total, blockIdx.x, shares);
    if (tid == 0) {
        to.total = total;
        to.shares = shares;
        to.placed = false;
        to.u = u;
        to.u_end = idle ? 0 : share_begin(total, blockIdx.x + 1, shares);
    }
    if (idle) return;
    if (one) {
        if (u >= upto - part && u < upto) to.b = tid, to.b_begin = upto - part;
        return;
    }
    long long before = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch && before <= u; b0 += THREADS) {
        const long long w = weight(b0 + tid);
        const long long end = inclusive(w) + before;
        if (u >= end - w && u < end) to.b = b0 + tid, to.b_begin = end - w;
        for (int x = 0; x < THREADS / 32; ++x) before += sum[x];
    }
}

// 16 consecutive elements of a query row as fp32.
template <typename T>
__device__ __forceinline__ void load_q16(float (&x)[16], const T *q, bool vec) {
    if (vec) {
        constexpr int N = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 16; i += N) {
            const uint4 u = *reinterpret_cast<const uint4 *>(q + i);
            const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
            for (int j = 0; j < N; ++j) x[i + j] = Elem<T>::to_float(e[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = Elem<T>::to_float(q[i]);
    }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(StreamCfg<D, NT>::kThreads, NT == 1 ? 2 : 1) paged_attention_stream_kernel(const __grid_constant__ StreamArgs sa) {
    using C = StreamCfg<D, NT>;
    constexpr int kStreamWarps = C::kWarps, kStreamThreads = C::kThreads, kTileKeys = C::kTileKeys;
    constexpr bool kSplit = sizeof(T) == 4;  // fp32 queries: two fp16 parts of q and of p
    constexpr int kParts = kSplit ? 2 : 1;
    constexpr int kSteps = D / 16;   // products of 16 along D
    constexpr int kHalves = D / 64;  // 16-byte loads of a key row
    constexpr int kMt = D / 16;      // 16-row tiles of O^T
    constexpr int kVBytes = D / 8;   // bytes of a V row a thread
    extern __shared__ __align__(16) uint8_t s_dyn[];
    float *const s_acc = reinterpret_cast<float *>(s_dyn + C::kDataBytes);
    __shared__ float s_m[kStreamWarps][C::kRows], s_l[kStreamWarps][C::kRows];
    __shared__ alignas(8) int s_lim[C::kRows];  // keys that a row sees
    __shared__ uint32_t s_nan[C::kRows][D / 32];  // columns of a row that are NaN, where s_any_nan
    __shared__ int s_any_nan;
    __shared__ long long s_sum[kStreamWarps];
    __shared__ Share s_share;
    __shared__ Segment s_segs[2];
    __shared__ bool s_more[2];
    __shared__ float s_qscale[C::kRows];  // raw product of a row to log2 units
    __shared__ long long s_to[C::kRows];  // where a row's output goes
    const AttnArgs &p = sa.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int group = p.H / p.Hkv;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    uint2 *const s_q = reinterpret_cast<uint2 *>(s_acc + C::kAccBytes / 4) + lane;  // [part][n][step][lane]

    if (tid == 0) sa.desc[blockIdx.x].segments = 0, s_any_nan = 0;
    for (int i = tid; i < C::kRows * (D / 32); i += kStreamThreads) s_nan[i / (D / 32)][i % (D / 32)] = 0;
    find_share<C::kRows, kTileKeys, C::kItemCost, kStreamThreads>(p, s_sum, s_share);
    __syncthreads();
    if (tid == 0) s_more[0] = next_segment<C::kRows, kTileKeys, C::kItemCost>(p, s_share, s_segs[0]);
    __syncthreads();

    // ---- this warp's keys: 16 of every tile, two tiles in shared memory, copied
    // there asynchronously; a table entry ahead of that.  16-byte chunks of a row
    // are exchanged by the row so that the reads below meet no bank twice: chunk c
    // of row r of the keys is at c ^ 4 (r % 2), of the values at c ^ 2 (r / 2 % 4)
    // (head size 128; at 64 the values' at c ^ (r / 2 % 4)).
    constexpr int kPerRow = D / 16, kCopies = D / 32;  // chunks of a row; copies a lane and side
    const uint32_t s_stage = static_cast<uint32_t>(__cvta_generic_to_shared(s_dyn)) + warp * 2 * C::kStageBytes;
    const int c_row = lane / kPerRow, c_chunk = lane % kPerRow;  // (rows c_row, c_row + 32 / kPerRow, ...)
    const int *entry = nullptr;  // of the table, of the next lookup
    int key = 0, key_end = 0, row = 0, ahead = -1;
    bool there = false, there_next = false;
    uint32_t stage = 0;
    const uint8_t *k_mine = nullptr, *v_mine = nullptr;
    const auto look_up = [&]() -> int { return __ldg(entry); };  // the table's entry of the next tile to copy
    // Copies the tile whose entry is x to stage st and steps on; true where its page is one.
    // (strides of the cache are below 2^31 bytes here, offsets 64-bit)
    const auto copy_tile = [&](int x, uint32_t st, const Segment &sg) -> bool {
        const bool ok = static_cast<unsigned>(x) < static_cast<unsigned>(p.num_blocks);
        if (ok) {
            const uint8_t *k = k_mine + static_cast<long long>(x) * sa.k_page + static_cast<long long>(row) * sa.k_row;
            const uint8_t *v = v_mine + static_cast<long long>(x) * sa.v_page + static_cast<long long>(row) * sa.v_row;
            const uint32_t to = s_stage + st * C::kStageBytes;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int r = c_row + i * (32 / kPerRow);
                copy16(to + r * D + (D == 128 ? (c_chunk ^ (r & 1) << 2) : c_chunk) * 16, k + i * (32 / kPerRow) * static_cast<long long>(sa.k_row));
                copy16(to + 16 * D + r * D + (D == 128 ? (c_chunk ^ (r >> 1 & 3) << 1) : (c_chunk ^ (r >> 1 & 3))) * 16,
                       v + i * (32 / kPerRow) * static_cast<long long>(sa.v_row));
            }
            if (lane < 2) copy4(to + 32 * D + lane * 4, (lane ? p.v.scale : p.k.scale) + x * p.Hkv + sg.h);
        }
        entry += sa.d_col;
        row += sa.d_row;
        if (row >= p.block) row -= p.block, ++entry;
        return ok;
    };
    const auto begin = [&](const Segment &sg) {  // the first copies of a segment
        key = sg.tile0 * kTileKeys + warp * 16;
        key_end = min(sg.tile1 * kTileKeys, sg.lim_max);
        const int col = key / p.block;
        row = key - col * p.block;
        entry = p.table + sg.b * p.table_stride + col;
        k_mine = p.k.base + sg.h * p.k.s[1] + c_row * p.k.s[2] + c_chunk * 16;
        v_mine = p.v.base + sg.h * p.v.s[1] + c_row * p.v.s[2] + c_chunk * 16;
        there = there_next = false;
        stage = 0;
        int x0 = -1, x1 = -1;
        if (key < key_end) x0 = look_up();
        if (key + kTileKeys < key_end) x1 = __ldg(entry + sa.d_col + (row + sa.d_row >= p.block ? 1 : 0));
        if (key < key_end) there = copy_tile(x0, 0, sg);
        copies_commit();
        if (key + kTileKeys < key_end) there_next = copy_tile(x1, 1, sg);
        copies_commit();
        if (key + 2 * kTileKeys < key_end) ahead = look_up();
    };

    // Query rows: warp n lays the n-th 8 out; it loads them as they are in memory
    // with the segment's first keys (rows of 16-byte vectors; others when laid out).
    constexpr int kQVecs = kHalves * sizeof(T);
    uint4 q_raw[kQVecs];
    const auto query_row = [&](const Segment &sg) -> const T * {
        const bool real = warp * 8 + g < sg.n_rows;
        const int rw = sg.row0 + warp * 8 + g, i = rw / group;
        return static_cast<const T *>(p.q) + (sg.r.first + (real ? i : 0)) * p.q_st[0] +
               (sg.h * group + (real ? rw - i * group : 0)) * p.q_st[1] + t * 16;
    };
    const auto begin_queries = [&](const Segment &sg) {
        if (warp >= NT || !sa.vec_q) return;
        const T *q = query_row(sg);
#pragma unroll
        for (int i = 0; i < kQVecs; ++i)
            q_raw[i] = *reinterpret_cast<const uint4 *>(q + i / static_cast<int>(sizeof(T)) * 64 +
                                                        i % static_cast<int>(sizeof(T)) * (16 / sizeof(T)));
    };

    if (s_more[0]) {
        begin(s_segs[0]);
        begin_queries(s_segs[0]);
    }
    for (int turn = 0; s_more[turn]; turn ^= 1) {
        const Segment &sg = s_segs[turn];
        // ---- the last warp walks on, the first ones lay the queries out as operands of S^T
        if (tid == kStreamThreads - 32)
            s_more[turn ^ 1] = next_segment<C::kRows, kTileKeys, C::kItemCost>(p, s_share, s_segs[turn ^ 1]);
        if (warp < NT) {
            const int n = warp;
            {
                const bool real = n * 8 + g < sg.n_rows;
                float x[kHalves][16];
                if (sa.vec_q) {
                    const T *y = reinterpret_cast<const T *>(q_raw);
#pragma unroll
                    for (int j = 0; j < kHalves * 16; ++j) x[j >> 4][j & 15] = Elem<T>::to_float(y[j]);
                } else {
                    const T *q = query_row(sg);
#pragma unroll
                    for (int j = 0; j < kHalves * 16; ++j)
                        x[j >> 4][j & 15] = Elem<T>::to_float(q[(j >> 4) * 64 + (j & 15)]);
                }
                float amax = 0.f;
#pragma unroll
                for (int j = 0; j < kHalves * 16; ++j) {
                    if (!real) x[j >> 4][j & 15] = 0.f;
                    amax = fmaxf(amax, fabsf(x[j >> 4][j & 15]));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const float c = p.scale * 1.4426950408889634f;
                const int e = query_exponent(amax, c);
                const float down = exp2_int(-e);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    uint2 hi, lo;
                    const float *y = &x[s >> 2][(s & 3) * 4];
                    hi.x = h2_bits(y[0] * down, y[1] * down);
                    hi.y = h2_bits(y[2] * down, y[3] * down);
                    s_q[(n * kSteps + s) * 32] = hi;
                    if constexpr (kSplit) {
                        const float2 h0 = h2_floats(hi.x), h1 = h2_floats(hi.y);
                        lo.x = h2_bits(y[0] * down - h0.x, y[1] * down - h0.y);
                        lo.y = h2_bits(y[2] * down - h1.x, y[3] * down - h1.y);
                        s_q[((NT + n) * kSteps + s) * 32] = lo;
                    }
                }
                if (t == 0) {
                    s_qscale[n * 8 + g] = exp2_int(e) * c;
                    s_lim[n * 8 + g] = real ? visible(p, sg.r, (sg.row0 + n * 8 + g) / group) : sg.r.keys;
                }
            }
        }
        __syncthreads();
        float acc[kMt][NT][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = kNoMax;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int x = 0; x < kMt; ++x) acc[x][n][0] = acc[x][n][1] = acc[x][n][2] = acc[x][n][3] = 0.f;
        }
        // (read in the loop, from shared memory: the registers are for the data)
        const volatile int &lim_min = sg.lim_min, &lim_max = sg.lim_max;
        const auto q_scale = [&](int n, int c) -> float {  // of column 2t + c
            return *static_cast<const volatile float *>(&s_qscale[n * 8 + 2 * t + c]);
        };
        for (; key < key_end; key += kTileKeys) {
            copies_wait_but_one();
            __syncwarp();
            const uint32_t at = s_stage + stage * C::kStageBytes;
            if (there) {
                // S^T: 16 keys, NT x 8 queries
                float s[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
                for (int hf = 0; hf < kHalves; ++hf) {
                    const int c = (hf * 4 + t) ^ (D == 128 ? (g & 1) << 2 : 0);
                    const uint4 k0 = shared16(at + g * D + c * 16), k8 = shared16(at + (g + 8) * D + c * 16);
                    const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w8[4] = {k8.x, k8.y, k8.z, k8.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a0 = e4m3x2_to_h2(w0[i]), a2 = e4m3x2_to_h2_hi(w0[i]);
                        const uint32_t a1 = e4m3x2_to_h2(w8[i]), a3 = e4m3x2_to_h2_hi(w8[i]);
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int part = 0; part < kParts; ++part) {
                                const uint2 q2 = s_q[((part * NT + n) * kSteps + hf * 4 + i) * 32];
                                mma16816(s[n], a0, a1, a2, a3, q2.x, q2.y);
                            }
                    }
                }
                const uint2 scales = shared8(at + 32 * D);
                const float ks = key_scale(__uint_as_float(scales.x)), vs = __uint_as_float(scales.y);
                const float vs_ok = value_scale(vs);
                const float lv = log2_fast(vs_ok), inv_vs = rcp_fast(vs_ok);
                const bool edge = key + 16 > lim_min;
                if (edge) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const int2 lim = *reinterpret_cast<const int2 *>(&s_lim[n * 8 + 2 * t]);
                        if (key + g >= lim.x) s[n][0] = -INFINITY;
                        if (key + g >= lim.y) s[n][1] = -INFINITY;
                        if (key + g + 8 >= lim.x) s[n][2] = -INFINITY;
                        if (key + g + 8 >= lim.y) s[n][3] = -INFINITY;
                    }
                }
                // w: the weight's exponent, value scale included.  Rounded before M is
                // taken from it: in one step the difference would keep the rounding of
                // M, which passes 1 where scores pass 2^24.
                bool raise = false;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float f0 = q_scale(n, 0) * ks, f1 = q_scale(n, 1) * ks;
                    s[n][0] = fmaf(s[n][0], f0, lv);
                    s[n][1] = fmaf(s[n][1], f1, lv);
                    s[n][2] = fmaf(s[n][2], f0, lv);
                    s[n][3] = fmaf(s[n][3], f1, lv);
                    raise = raise || fmaxf(s[n][0], s[n][2]) - m[n][0] > kTopExp || fmaxf(s[n][1], s[n][3]) - m[n][1] > kTopExp;
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float top = fmaxf(s[n][c], s[n][c + 2]);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            top = fmaxf(top - kLift<T>, m[n][c]);
                            const float half = exp2_half(m[n][c] - top), fix = half * half;
                            m[n][c] = top;
                            l[n][c] = l[n][c] * half * half;
#pragma unroll
                            for (int x = 0; x < kMt; ++x) acc[x][n][c] *= fix, acc[x][n][c + 2] *= fix;
                        }
                }
                uint32_t pf[kParts][NT][2];  // P^T, keys along the operand's rows
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float p0 = exp2_fast(s[n][0] - m[n][0]), p1 = exp2_fast(s[n][1] - m[n][1]);
                    const float p2 = exp2_fast(s[n][2] - m[n][0]), p3 = exp2_fast(s[n][3] - m[n][1]);
                    if (lv < kSmallScale) {
                        l[n][0] += exp2_fast(s[n][0] - m[n][0] - lv) + exp2_fast(s[n][2] - m[n][0] - lv);
                        l[n][1] += exp2_fast(s[n][1] - m[n][1] - lv) + exp2_fast(s[n][3] - m[n][1] - lv);
                    } else {
                        l[n][0] = fmaf(p0 + p2, inv_vs, l[n][0]);
                        l[n][1] = fmaf(p1 + p3, inv_vs, l[n][1]);
                    }
                    const uint32_t a = h2_bits(p0, p1), c = h2_bits(p2, p3);
                    pf[0][n][0] = transpose8x8(a);
                    pf[0][n][1] = transpose8x8(c);
                    if constexpr (kSplit) {
                        const float2 ah = h2_floats(a), ch = h2_floats(c);
                        pf[kParts - 1][n][0] = transpose8x8(h2_bits(p0 - ah.x, p1 - ah.y));
                        pf[kParts - 1][n][1] = transpose8x8(h2_bits(p2 - ch.x, p3 - ch.y));
                    }
                }
                uint32_t vr[4][kVBytes / 4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = 2 * t + (i & 1) + (i >> 1) * 8;
                    const uint32_t v_at = at + 16 * D + r * D;
                    if constexpr (D == 128) {
                        const uint4 x = shared16(v_at + (g ^ t << 1) * 16);
                        vr[i][0] = x.x, vr[i][1] = x.y, vr[i][kVBytes / 4 - 2] = x.z, vr[i][kVBytes / 4 - 1] = x.w;
                    } else {
                        const uint2 x = shared8(v_at + ((g >> 1) ^ t) * 16 + (g & 1) * 8);
                        vr[i][0] = x.x, vr[i][1] = x.y;
                    }
                }
                if (edge) {
                    // Rows behind the last key: zero.
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key + 2 * t + (i & 1) + (i >> 1) * 8 >= lim_max)
#pragma unroll
                            for (int x = 0; x < kVBytes / 4; ++x) vr[i][x] = 0;
                    // NaN in rows that some queries do not see.
                    uint32_t nan = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int x = 0; x < kVBytes / 4; ++x) nan |= nan_bits(vr[i][x]);
                    if (__any_sync(0xffffffffu, nan != 0)) {
                        if (lane < sg.n_rows) mark_nan(p, p.table + sg.b * p.table_stride, sg.h, key, min(key + 16, s_lim[lane]), s_nan[lane]);
                        if (lane == 0) s_any_nan = 1;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int x = 0; x < kVBytes / 4; ++x) vr[i][x] = without_nan(vr[i][x]);
                    }
                }
                // O^T += V^T P^T
#pragma unroll
                for (int x = 0; x < kVBytes / 4; ++x) {
                    const uint32_t e0 = __byte_perm(vr[0][x], vr[1][x], 0x5140);  // dims 4x, 4x + 1 of keys 2t, 2t + 1
                    const uint32_t o0 = __byte_perm(vr[0][x], vr[1][x], 0x7362);  // dims 4x + 2, 4x + 3
                    const uint32_t e1 = __byte_perm(vr[2][x], vr[3][x], 0x5140);  // of keys 2t + 8, 2t + 9
                    const uint32_t o1 = __byte_perm(vr[2][x], vr[3][x], 0x7362);
                    const uint32_t a0 = e4m3x2_to_h2(e0), a1 = e4m3x2_to_h2_hi(e0);
                    const uint32_t a2 = e4m3x2_to_h2(e1), a3 = e4m3x2_to_h2_hi(e1);
                    const uint32_t c0 = e4m3x2_to_h2(o0), c1 = e4m3x2_to_h2_hi(o0);
                    const uint32_t c2 = e4m3x2_to_h2(o1), c3 = e4m3x2_to_h2_hi(o1);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int part = 0; part < kParts; ++part) {
                            mma16816(acc[2 * x][n], a0, a1, a2, a3, pf[part][n][0], pf[part][n][1]);
                            mma16816(acc[2 * x + 1][n], c0, c1, c2, c3, pf[part][n][0], pf[part][n][1]);
                        }
                }
            }
            __syncwarp();  // the stage has been read
            bool more = false;
            if (key + 2 * kTileKeys < key_end) more = copy_tile(ahead, stage, sg);
            copies_commit();
            there = there_next;
            there_next = more;
            stage ^= 1;
            if (key + 3 * kTileKeys < key_end) ahead = look_up();
        }

        // ---- the next segment's first copies, then the warps join
        if (s_more[turn ^ 1]) begin(s_segs[turn ^ 1]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
                if (g == 0) {
                    s_m[warp][n * 8 + 2 * t + c] = m[n][c];
                    s_l[warp][n * 8 + 2 * t + c] = l[n][c];
                }
            }
        const bool whole = sg.tile0 == 0 && sg.tile1 == sg.tiles;
        const int slot = 2 * blockIdx.x + (sg.tile0 == 0 ? 1 : 0);
        // The rows' own: each warp's weight, 1 / sum in it, and where the row goes.
        const auto join_rows = [&]() {
            if (tid >= sg.n_rows) return;
            const int rw = tid;
            float top = s_m[0][rw];
#pragma unroll
            for (int w = 1; w < kStreamWarps; ++w) top = fmaxf(top, s_m[w][rw]);
            // (a warp that saw no key adds nothing: its l and sums are 0)
            float sum = 0.f, fix[kStreamWarps];
#pragma unroll
            for (int w = 0; w < kStreamWarps; ++w) {
                const float half = exp2_half(s_m[w][rw] - top);
                fix[w] = half * half;
                sum = fmaf(half, half * s_l[w][rw], sum);
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int w = 0; w < kStreamWarps; ++w) s_m[w][rw] = fix[w] * inv;
            const float lse2 = sum == 0.f ? -INFINITY : top + log2f(sum);
            if (whole) {
                const int tok = (sg.row0 + rw) / group, head = sg.h * group + (sg.row0 + rw) - tok * group;
                const long long token = sg.r.first + tok;
                s_to[rw] = token * p.o_st[0] + head * p.o_st[1];
                if (p.lse) p.lse[token * p.H + head] = lse2 * 0.6931471805599453f;
            } else {
                s_to[rw] = (static_cast<long long>(slot) * C::kRows + rw) * D;
                sa.part_lse[slot * C::kRows + rw] = lse2;
            }
        };
        // A warp's sums, times its weights where two warps share a place.
        constexpr bool kTwoRounds = C::kSlots < kStreamWarps;
        const auto store_sums = [&](bool add) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int rw = n * 8 + 2 * t + c;
                    if (rw >= sg.n_rows) continue;
                    const float fix = kTwoRounds ? s_m[warp][rw] : 1.f;
                    float4 *to = reinterpret_cast<float4 *>(s_acc + (warp % C::kSlots * C::kRows + rw) * C::kRowPitch + g * (D / 8 + 4));
#pragma unroll
                    for (int x = 0; x < kMt / 2; ++x) {
                        float4 v = make_float4(acc[2 * x][n][c] * fix, acc[2 * x][n][c + 2] * fix, acc[2 * x + 1][n][c] * fix,
                                               acc[2 * x + 1][n][c + 2] * fix);
                        if (add) {
                            const float4 o = to[x];
                            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
                        }
                        to[x] = v;
                    }
                }
        };
        if constexpr (!kTwoRounds) store_sums(false);
        if (s_more[turn ^ 1]) begin_queries(s_segs[turn ^ 1]);
        __syncthreads();
        if constexpr (kTwoRounds) {
            join_rows();
            __syncthreads();
            if (warp < C::kSlots) store_sums(false);
            __syncthreads();
            if (warp >= C::kSlots) store_sums(true);
            __syncthreads();
            // Four columns of a row a thread.
            for (int i = tid; i < sg.n_rows * (D / 4); i += kStreamThreads) {
                const int rw = i / (D / 4), d = i % (D / 4) * 4;
                const float *from = s_acc + rw * C::kRowPitch + d + d / (D / 8) * 4;
                float x[4] = {};
#pragma unroll
                for (int w = 0; w < C::kSlots; ++w) {
                    const float4 v = *reinterpret_cast<const float4 *>(from + w * C::kRows * C::kRowPitch);
                    x[0] += v.x, x[1] += v.y, x[2] += v.z, x[3] += v.w;
                }
                if (s_any_nan) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (s_nan[rw][d >> 5] >> ((d & 31) + c) & 1u) x[c] = NAN;
                }
                if (whole) {
                    T *o = static_cast<T *>(p.o) + s_to[rw] + d;
                    alignas(16) T y[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) y[c] = Elem<T>::from_float(x[c]);
                    if (sa.vec_o) {
                        if constexpr (sizeof(T) == 4)
                            *reinterpret_cast<uint4 *>(o) = *reinterpret_cast<const uint4 *>(y);
                        else
                            *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<const uint2 *>(y);
                    } else {
#pragma unroll
                        for (int c = 0; c < 4; ++c) o[c] = y[c];
                    }
                } else {
                    *reinterpret_cast<float4 *>(sa.part_o + s_to[rw] + d) = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
        } else {
            // Few rows: each thread weighs the warps for its own column (one barrier less;
            // 2 x 128 keys 6.1 us against 6.8 with the rows' weights formed once).
            for (int i = tid; i < sg.n_rows * D; i += kStreamThreads) {
                const int rw = i / D, d = i - rw * D;
                const float *from = s_acc + rw * C::kRowPitch + d + d / (D / 8) * 4;
                float top = s_m[0][rw];
#pragma unroll
                for (int w = 1; w < kStreamWarps; ++w) top = fmaxf(top, s_m[w][rw]);
                // (a warp that saw no key adds nothing: its l and sums are 0)
                float sum = 0.f, x = 0.f;
#pragma unroll
                for (int w = 0; w < kStreamWarps; ++w) {
                    const float half = exp2_half(s_m[w][rw] - top);
                    sum = fmaf(half, half * s_l[w][rw], sum);
                    x = fmaf(half * half, from[w * C::kRows * C::kRowPitch], x);
                }
                x *= sum == 0.f ? 0.f : 1.f / sum;
                if (s_any_nan && (s_nan[rw][d >> 5] >> (d & 31) & 1u)) x = NAN;
                const float lse2 = sum == 0.f ? -INFINITY : top + log2f(sum);
                if (whole) {
                    const int tok = (sg.row0 + rw) / group, head = sg.h * group + (sg.row0 + rw) - tok * group;
                    const long long token = sg.r.first + tok;
                    static_cast<T *>(p.o)[token * p.o_st[0] + head * p.o_st[1] + d] = Elem<T>::from_float(x);
                    if (p.lse && d == 0) p.lse[token * p.H + head] = lse2 * 0.6931471805599453f;
                } else {
                    sa.part_o[(static_cast<long long>(slot) * C::kRows + rw) * D + d] = x;
                    if (d == 0) sa.part_lse[slot * C::kRows + rw] = lse2;
                }
            }
        }
        if (tid == 0 && sg.tile0 == 0 && !whole)  // begun here, ended by a later CTA
            sa.desc[blockIdx.x] = StreamDesc{sg.last_cta - static_cast<int>(blockIdx.x) + 1, sg.r.first, sg.h, sg.row0, sg.n_rows, {}};
        if (s_any_nan) {
            __syncthreads();
            for (int i = tid; i < C::kRows * (D / 32); i += kStreamThreads) s_nan[i / (D / 32)][i % (D / 32)] = 0;
            __syncthreads();
            if (tid == 0) s_any_nan = 0;
        }
        __syncthreads();  // the queries, sums and segment may be written over
    }
    clear_unused<T>(p);
}

// Joins the partial rows of the item that CTA blockIdx.x of the kernel before
// began and did not end: a warp a row, each lane D / 32 neighbouring columns.
constexpr int kJoinThreads = 256;

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) paged_attention_join_kernel(const __grid_constant__ StreamArgs sa) {
    constexpr int kCols = D / 32;
    const AttnArgs &p = sa.a;
    const int lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const StreamDesc desc = sa.desc[blockIdx.x];
    const int n = desc.segments, rw = blockIdx.y * (kJoinThreads / 32) + (threadIdx.x >> 5);
    if (n == 0 || rw >= desc.n_rows) return;
    // Part i lies in slot 2c + 1 of the CTA that began the item (i = 0), in slot 2c of those after it.
    const auto slot = [&](int i) { return i == 0 ? 2 * static_cast<int>(blockIdx.x) + 1 : 2 * (static_cast<int>(blockIdx.x) + i); };
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) top = fmaxf(top, sa.part_lse[slot(i) * ROWS + rw]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x[kCols] = {};
    for (int i0 = 0; i0 < n; i0 += 32) {
        const float w = i0 + lane < n ? exp2_fast(sa.part_lse[slot(i0 + lane) * ROWS + rw] - base) : 0.f;
        sum += w;
        const int here = min(32, n - i0);
#pragma unroll 8
        for (int i = 0; i < here; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const float *from = sa.part_o + (static_cast<long long>(slot(i0 + i)) * ROWS + rw) * D + lane * kCols;
            if constexpr (kCols == 4) {
                const float4 v = *reinterpret_cast<const float4 *>(from);
                x[0] = fmaf(wi, v.x, x[0]), x[1] = fmaf(wi, v.y, x[1]), x[2] = fmaf(wi, v.z, x[2]), x[3] = fmaf(wi, v.w, x[3]);
            } else {
                const float2 v = *reinterpret_cast<const float2 *>(from);
                x[0] = fmaf(wi, v.x, x[0]), x[1] = fmaf(wi, v.y, x[1]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int group = p.H / p.Hkv, row = desc.row0 + rw, tok = row / group, head = desc.h * group + row - tok * group;
    const long long token = desc.first + tok;
    T *o = static_cast<T *>(p.o) + token * p.o_st[0] + head * p.o_st[1] + lane * kCols;
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c] = Elem<T>::from_float(x[c] * inv);
    if (p.lse && lane == 0)
        p.lse[token * p.H + head] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.6931471805599453f;
}

}  // namespace paged
}  // namespace pmkl_b200
