// paged_attention_tile.cuh -- attention of many query rows a request over the
// paged 8-bit cache on the tcgen05 tensor cores: fp16/bf16 queries, head size
// 64 or 128, pages of a multiple of 16 rows.
//
// The rows that read one K/V head (tokens times the group's query heads) are
// taken 128 at a time, and the list of (request, K/V head, row tile) items, cut
// in tiles of 128 keys, is shared out evenly over resident CTAs as in the
// stream kernel; a row tile's key tiles end with the last key that it sees.
//
// A CTA has three warpgroups, which divide its registers between them
// (setmaxnreg); two CTAs an SM fill each other's gaps:
//   * warps 4, 5 bring keys in, warps 6, 7 values: 8-bit values loaded 16 bytes a thread, half a tile ahead in registers, made fp16
//     (every e4m3 value is one) and stored as the 128-byte-swizzled tiles that
//     the products read.  No scale is multiplied in: they go with the scores;
//   * warp 10 looks the tiles' pages up: addresses and scales;
//   * warp 9 walks the CTA's share and hands out its segments;
//   * warp 8 issues tcgen05.mma: S = Q K^T, then O += P V with P from tensor
//     memory.  Products of one thread run in order, so S of the next tile may
//     be issued over P, and its completion tells that P V is done;
//   * warps 0-3, a thread a row: the running maximum and sum.  A page's key
//     scale and the row's factor make one factor for 16 scores, its value scale
//     enters the exponent; weights go up to 2^15, and the reference is raised, and
//     O rescaled, only when one would pass that (as in the stream kernel).  They
//     also load the queries and write the results.  Score and reference meet in
//     one multiply-add, which is exact enough while the reference is below 2^20;
//     beyond, the exponents are formed in two steps beforehand (two steps for all:
//     498 us against 476 on the chunks below), as they are where a page's value
//     scale is small and far below one before it (715 us on the chunks).  What is seldom needed (masks,
//     rescaling, those exponents) goes through tensor memory in rolled loops: the
//     warps' code has to stay in the instruction cache (masks in registers and
//     an unrolled rescaling, 5 KB more: prompts of 1000 tokens 489 us against 461).
// Tensor memory (256 columns a CTA): S [0, 128), O [128, 128 + D); P takes S's
// upper half: scores 64..127 are held in registers when it is written.
//
// What bounds it: each CTA's chain (S 600 cycles, softmax 3300, P V 600, and the
// hand-overs), some 6000 cycles a tile with two CTAs an SM, against 1024 cycles
// of tensor work.  B200, device time: chunks of 700..1024 tokens over 3001..8192
// keys, 32/8 heads of 128 (bf16): 478 us, 622 TFLOP/s (0.38 of the measured bf16
// rate); 1..5 tokens over 500..8192 keys, 32/4 heads (fp16): 53 us, where the
// loads' latency is the chain (a half tile of keys and one of values a CTA under
// way).
// Tried and not kept: weights against the last reference with a second pass
// where the maximum passes it (P would wait in registers: spills); one CTA an SM
// (1098 us against 736 at that step).
//
// NaN and rows behind the last key: as in the stream kernel.  Values in tiles
// at the diagonal are searched for NaN; where there is one, the product gets
// zeros and the rows that see the key note its columns.
#pragma once

#include "paged_attention_stream.cuh"
#include "sm100_ptx.cuh"

namespace pmkl_b200 {
namespace paged {

constexpr int kTileRows = 128;
constexpr int kTileThreads = 384;
constexpr int kTileItemCost = 1;  // of an item, in tiles: some 8000 cycles against 7000
// Registers a thread: at launch, and what each warpgroup sets; the three come
// to the launch's total (the host checks that the build has it).  B200, chunk
// workload above: 120/64/56 and 120/72/48 481 us, 112/72/56 492, 128/72/40 564,
// 128/80/32 653; 16 x 1..5 tokens: 52.7, 54.4, 55.2, 62, 68.5.
constexpr int kTileLaunchRegs = 80, kTileSoftmaxRegs = 120, kTileLoadRegs = 64, kTileIssueRegs = 56;
static_assert(kTileSoftmaxRegs + kTileLoadRegs + kTileIssueRegs == 3 * kTileLaunchRegs, "register split");
constexpr int kMaxTileCtas = 320;  // partials in the workspace: 148 SMs with 2 CTAs

// A warpgroup's share; only the matching direction is allowed.
template <int N>
__device__ __forceinline__ void set_regs() {
    if constexpr (N < kTileLaunchRegs)
        ptx::reg_dealloc<N>();
    else
        ptx::reg_alloc<N>();
}

template <int D>
struct TileCfg {
    static constexpr int kBoxes = D / 64;
    static constexpr int kTileBytes = kBoxes * 128 * 128;
    static constexpr int kSmemBytes = 3 * kTileBytes + 1024;
    static constexpr uint32_t kTmemCols = 256, kColS = 0, kColP = 64, kColO = 128;
};

constexpr int kAhead = 4;

// Powers of two that a value scale lies below the segment's largest so far, from
// which on the sum's terms come from exponents of their own (kSmallScale, but
// pages of zeros, whose scale is 2^-64, are then seldom among them).
constexpr float kFarScale = 64.f;

// References up to here: what the multiply-add of a score with its reference may
// be off, four roundings of it, stays below 2^-2 (weights below fp16's largest).
constexpr float kExactRef = 1048576.f;

struct TileShared {
    uint64_t q_full, k_full, k_empty, v_full, v_empty, s_full, p_full, o_full, drained;
    uint64_t seg_full[2], seg_empty[2], page_full[kAhead], page_empty[kAhead];
    uint32_t tmem;
    int abort_flag;
    Share share;
    Segment seg[2];
    // Of four tiles' groups of 16 keys: where they begin (0: no page) in the keys
    // and the values; key scale, log2 of the value scale (-inf: no page).
    unsigned long long from[kAhead][2][8];
    // The last: (1, 0) and 0, for scores that are exponents already.
    float2 scale[kAhead + 1][8];
    float inv_vs[kAhead + 1][8];
    int small[kAhead];   // some group's value scale is small beside the segment's largest so far
    int nan[2];          // the tile's values held NaN: tile number of the CTA + 1
    alignas(16) uint32_t nan_cols[kTileRows][4];  // columns of a row that are NaN (see above)
    long long sum[kTileThreads / 32];
};

// tcgen05.wait::ld that the values pass through, so that no use of them is
// moved before it.
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15])
                 :
                 : "memory");
    asm volatile(""
                 : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// Bounded wait of a whole warp, every lane testing and all of one answer; a
// rolled loop, as the kernel's code has to stay in the instruction cache.
__device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
    const unsigned long long t0 = ptx::globaltimer();
#pragma unroll 1
    for (;;) {
        if (__all_sync(0xffffffffu, ptx::mbar_try_wait_suspend(bar, parity))) return true;
        if (ptx::globaltimer() - t0 > ptx::kWaitTimeoutNs) *abort_flag = 1;
        if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
    }
}

// 16 columns, waited for.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// Largest of 16 scores.
__device__ __forceinline__ float max16(const uint32_t *r) {
    float m = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
#pragma unroll
    for (int i = 2; i < 16; i += 2) m = ptx::fmax3(m, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    return m;
}

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 2) paged_attention_tile_kernel(const __grid_constant__ StreamArgs sa) {
    using namespace ptx;
    using C = TileCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ TileShared sh;
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *sQ = smem, *sK = smem + C::kTileBytes, *sV = smem + 2 * C::kTileBytes;
    const AttnArgs &p = sa.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = p.H / p.Hkv;
    volatile int *abort_flag = &sh.abort_flag;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // ---- set-up: barriers, tensor memory, this CTA's share
    if (tid == 0) {
        mbar_init(&sh.q_full, 128);
        mbar_init(&sh.k_full, 64);
        mbar_init(&sh.k_empty, 1);
        mbar_init(&sh.v_full, 64);
        mbar_init(&sh.v_empty, 1);
        mbar_init(&sh.s_full, 1);
        mbar_init(&sh.p_full, 128);
        mbar_init(&sh.o_full, 1);
        mbar_init(&sh.drained, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.seg_full[i], 1);
            mbar_init(&sh.seg_empty[i], 10);  // four softmax and four loading warps, two of the third group
        }
        for (int i = 0; i < kAhead; ++i) {
            mbar_init(&sh.page_full[i], 1);
            mbar_init(&sh.page_empty[i], 8);  // four softmax and four loading warps
        }
        sh.nan[0] = sh.nan[1] = 0;
        for (int i = 0; i < 8; ++i) sh.scale[kAhead][i] = make_float2(1.f, 0.f), sh.inv_vs[kAhead][i] = 0.f;
        // Once any CTA has given up a wait, later CTAs skip their work.
        sh.abort_flag = (*reinterpret_cast<volatile unsigned int *>(&g_device_error) != 0u) ? 1 : 0;
        sa.desc[blockIdx.x].segments = 0;
        fence_mbarrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&sh.tmem, C::kTmemCols);
        tmem_relinquish();
    }
    find_share<kTileRows, 128, kTileItemCost, kTileThreads>(p, sh.sum, sh.share);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const bool skip = *abort_flag != 0;
    if (warp >= 8) {
        // ------------------------------------------------------------ products
        set_regs<kTileIssueRegs>();
        if (warp == 9 && lane == 0 && !skip) {
            // The segments, two ahead at most; one without tiles is the end.
            bool more = true;
            for (uint32_t seg = 0; more; ++seg) {
                const int i = seg & 1;
                if (seg >= 2 && !mbar_wait(&sh.seg_empty[i], ((seg >> 1) - 1) & 1, abort_flag)) break;
                Segment &s = sh.seg[i];
                more = next_segment<kTileRows, 128, kTileItemCost>(p, sh.share, s);
                if (!more) s.tile0 = s.tile1 = 0;
                mbar_arrive(&sh.seg_full[i]);
            }
        }
        else if (warp == 10 && !skip) {
            // The tiles' pages: addresses and scales, up to four tiles ahead.
            const CacheView &cache = lane < 8 ? p.k : p.v;
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t seg = 0; ok; ++seg) {
                if (!(ok = wait_warp(&sh.seg_full[seg & 1], (seg >> 1) & 1, abort_flag))) break;
                const Segment &s = sh.seg[seg & 1];
                const int *table = p.table + s.b * p.table_stride;
                const int tile0 = s.tile0, tile1 = s.tile1, lim_max = s.lim_max, h = s.h;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.seg_empty[seg & 1]);
                if (tile0 == tile1) break;
                const auto look_up = [&](int j) {
                    const int key = j * 128 + (lane & 7) * 16;
                    return key < lim_max ? __ldg(table + key / p.block) : -1;
                };
                int x = look_up(tile0);
                float lv_top = -INFINITY;  // the largest log2 of a value scale so far
                for (int j = tile0; j < tile1; ++j, ++it) {
                    const int x_next = j + 1 < tile1 ? look_up(j + 1) : -1;
                    const int row = (j * 128 + (lane & 7) * 16) % p.block;
                    unsigned long long from = 0;
                    float ks = 1.f, vs = 1.f;  // no page: any key scale but 0, for masked scores are -inf
                    const bool there = x >= 0 && x < p.num_blocks;
                    if (there) {
                        from = reinterpret_cast<unsigned long long>(cache.base) + x * cache.s[0] + h * cache.s[1] +
                               row * cache.s[2];
                        const long long at = static_cast<long long>(x) * p.Hkv + h;
                        ks = key_scale(__ldg(p.k.scale + at));
                        vs = value_scale(__ldg(p.v.scale + at));
                    }
                    const float lv = there ? log2f(vs) : -INFINITY;
                    lv_top = fmaxf(lv_top, lv);
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) lv_top = fmaxf(lv_top, __shfl_xor_sync(0xffffffffu, lv_top, o));
                    const int small = __any_sync(0xffffffffu, there && lv_top - lv > kFarScale);
                    const int i = it % kAhead;
                    if (it >= kAhead && !(ok = wait_warp(&sh.page_empty[i], (it / kAhead - 1) & 1, abort_flag))) break;
                    if (lane < 16) sh.from[i][lane >> 3][lane & 7] = from;
                    if (lane < 8) {
                        sh.scale[i][lane] = make_float2(ks, lv);
                        sh.inv_vs[i][lane] = 1.f / vs;
                    }
                    if (lane == 0) sh.small[i] = small;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.page_full[i]);
                    x = x_next;
                }
            }
        }
        else if (warp == 8 && lane == 0 && !skip) {
            constexpr uint32_t kIdescS = idesc_f16(128, 128, 0, 0, 0);
            constexpr uint32_t kIdescO = idesc_f16(128, D, 0, 0, 1);
            const uint64_t q_desc = smem_desc_sw128(smem_u32(sQ), 16, 1024), k_desc = smem_desc_sw128(smem_u32(sK), 16, 1024);
            const uint64_t v_desc = smem_desc_sw128(smem_u32(sV), 128 * 128, 1024);
            // The halves: addresses advance in the low one, in units of 16 bytes.
            const uint32_t q_lo = static_cast<uint32_t>(q_desc), k_lo = static_cast<uint32_t>(k_desc);
            const uint32_t v_lo = static_cast<uint32_t>(v_desc);
            const uint32_t qk_hi = static_cast<uint32_t>(q_desc >> 32), v_hi = static_cast<uint32_t>(v_desc >> 32);
            uint32_t it = 0;
            bool ok = true;
            for (uint32_t seg = 0; ok; ++seg) {
                if (!(ok = mbar_wait(&sh.seg_full[seg & 1], (seg >> 1) & 1, abort_flag))) break;
                int tiles = sh.seg[seg & 1].tile1 - sh.seg[seg & 1].tile0;
                mbar_arrive(&sh.seg_empty[seg & 1]);
                if (tiles == 0) break;
                ok = mbar_wait(&sh.q_full, seg & 1, abort_flag);
                for (uint32_t more = 0; ok && tiles > 0; --tiles, ++it, more = 1) {
                    if (!(ok = mbar_wait(&sh.k_full, it & 1, abort_flag))) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = ((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4;
                        mma_ss_h(tmem + C::kColS, q_lo + off, qk_hi, k_lo + off, qk_hi, kIdescS, kk > 0 ? 1u : 0u);
                    }
                    mma_commit(&sh.s_full);
                    mma_commit(&sh.k_empty);
                    if (!(ok = mbar_wait(&sh.v_full, it & 1, abort_flag))) break;
                    if (!(ok = mbar_wait(&sh.p_full, it & 1, abort_flag))) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk)
                        mma_ts_h(tmem + C::kColO, tmem + C::kColP + kk * 8, v_lo + kk * (16 * 128 / 16), v_hi, kIdescO,
                                 kk > 0 ? 1u : more);
                    mma_commit(&sh.v_empty);
                }
                if (ok) mma_commit(&sh.o_full);
            }
            // Every product has ended before tensor memory is given back.
            mma_commit(&sh.drained);
            volatile int never = 0;
            mbar_wait(&sh.drained, 0, &never);
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------ cache to shared memory
        set_regs<kTileLoadRegs>();
        constexpr int kPerRow = D / 16;          // threads a row, 16 bytes each
        constexpr int kRowsPass = 64 / kPerRow;  // rows a pass: 8 or 16
        constexpr int kHalf = 64 / kRowsPass;    // passes of half a tile
        const bool values = warp >= 6;
        const CacheView &cache = values ? p.v : p.k;
        uint64_t *const full = values ? &sh.v_full : &sh.k_full, *const empty = values ? &sh.v_empty : &sh.k_empty;
        const int t = tid & 63, chunk = t % kPerRow;
        // Threads of the second 64 columns take the row next to it: the eight
        // that store at one time then meet all banks once.
        const int sub = (t / kPerRow) ^ (chunk >> 2);
        uint8_t *const to = (values ? sV : sK) + (chunk >> 2) * (128 * 128) + sub * 128;
        const int at0 = (((chunk & 3) * 2) ^ (sub & 7)) << 4, at1 = (((chunk & 3) * 2 + 1) ^ (sub & 7)) << 4;
        const long long row_bytes = cache.s[2], mine_off = sub * row_bytes + chunk * 16, mine_odd = mine_off + 8 * row_bytes;
        uint32_t it = 0;
        bool ok = !skip;
        for (uint32_t seg = 0; ok; ++seg) {
            if (!(ok = wait_warp(&sh.seg_full[seg & 1], (seg >> 1) & 1, abort_flag))) break;
            const Segment &s = sh.seg[seg & 1];
            const int tile0 = s.tile0, tile1 = s.tile1, lim_min = s.lim_min, lim_max = s.lim_max;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.seg_empty[seg & 1]);
            if (tile0 == tile1) break;
            uint4 v[kHalf];
            // Half a tile, 64 rows, into registers; rows that no query sees, or in no
            // page of the cache, are zero.  `n`: the CTA's tile number.
            const auto load = [&](int f, uint32_t n) {
                const int i_page = n % kAhead;
                if (!(f & 1) && !(ok = wait_warp(&sh.page_full[i_page], n / kAhead & 1, abort_flag))) return;
                const unsigned long long *from = &sh.from[i_page][values ? 1 : 0][(f & 1) * 4];
                const int left = lim_max - f * 64 - sub;
#pragma unroll
                for (int i = 0; i < kHalf; ++i) {
                    const unsigned long long at = from[i * kRowsPass / 16];
                    v[i] = load16_if(reinterpret_cast<const uint8_t *>(at) + (i * kRowsPass % 16 ? mine_odd : mine_off),
                                     at != 0 && i * kRowsPass < left);
                }
                if (f & 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.page_empty[i_page]);
                }
            };
            load(2 * tile0, it);
            for (int f = 2 * tile0; ok && f < 2 * tile1; ++f) {
                const bool second = f & 1;
                if (!second && it > 0 && !(ok = wait_warp(empty, (it - 1) & 1, abort_flag))) break;
                uint8_t *const here = to + (second ? 64 * 128 : 0);
#pragma unroll
                for (int i = 0; i < kHalf; ++i) {
                    *reinterpret_cast<uint4 *>(here + i * (kRowsPass * 128) + at0) =
                        make_uint4(e4m3x2_to_h2(v[i].x), e4m3x2_to_h2_hi(v[i].x), e4m3x2_to_h2(v[i].y),
                                   e4m3x2_to_h2_hi(v[i].y));
                    *reinterpret_cast<uint4 *>(here + i * (kRowsPass * 128) + at1) =
                        make_uint4(e4m3x2_to_h2(v[i].z), e4m3x2_to_h2_hi(v[i].z), e4m3x2_to_h2(v[i].w),
                                   e4m3x2_to_h2_hi(v[i].w));
                }
                if (values && f * 64 + 64 > lim_min) {
                    // NaN among the values: noted, and zero in the tile.
                    uint32_t nan = 0;
#pragma unroll
                    for (int i = 0; i < kHalf; ++i)
                        nan |= nan_bits(v[i].x) | nan_bits(v[i].y) | nan_bits(v[i].z) | nan_bits(v[i].w);
                    if (nan) {
                        sh.nan[it & 1] = static_cast<int>(it) + 1;
#pragma unroll 1
                        for (int i = 0; i < kHalf * 16; ++i) {
                            uint16_t *x = reinterpret_cast<uint16_t *>(here + (i >> 4) * (kRowsPass * 128) +
                                                                       ((i & 8) ? at1 : at0)) + (i & 7);
                            if ((*x & 0x7FFF) > 0x7C00) *x = 0;
                        }
                    }
                }
                if (second) {
                    fence_proxy_async_smem();
                    mbar_arrive(full);
                    ++it;
                }
                if (f + 1 < 2 * tile1) load(f + 1, it);
            }
        }
    } else {
        // ------------------------------------------------------------ softmax, a thread a row
        set_regs<kTileSoftmaxRegs>();
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
        uint32_t it = 0;
        bool ok = !skip;
        for (uint32_t seg = 0; ok; ++seg) {
            if (!(ok = wait_warp(&sh.seg_full[seg & 1], (seg >> 1) & 1, abort_flag))) break;
            const Segment &s = sh.seg[seg & 1];
            const int tile0 = s.tile0, tile1 = s.tile1, lim_min = s.lim_min;
            if (tile0 == tile1) break;
            const int rr = s.row0 + tid;
            const bool real = tid < s.n_rows;
            const int tok = real ? rr / group : 0, head = s.h * group + (real ? rr - tok * group : 0);
            const T *q = static_cast<const T *>(p.q) + (s.r.first + tok) * p.q_st[0] + head * p.q_st[1];
            // The row's largest value, then the row over its power of two.
            float amax = 0.f;
            if (real)
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    float x[16];
                    load_q16(x, q + c, sa.vec_q != 0);
#pragma unroll
                    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
                }
            const float log2_scale = p.scale * 1.4426950408889634f;
            const int e = query_exponent(amax, log2_scale);
            const float down = exp2_int(-e);
            const float row_up = exp2_int(e) * log2_scale;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                float x[16];
                if (real) load_q16(x, q + c, sa.vec_q != 0);
                uint32_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = real ? h2_bits(x[2 * i] * down, x[2 * i + 1] * down) : 0u;
                uint8_t *box = sQ + (c >> 6) * (128 * 128) + tid * 128;
                const int at = (c & 63) >> 3;
                *reinterpret_cast<uint4 *>(box + (((at) ^ (tid & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                *reinterpret_cast<uint4 *>(box + (((at + 1) ^ (tid & 7)) << 4)) = make_uint4(w[4], w[5], w[6], w[7]);
            }
            fence_proxy_async_smem();
            mbar_arrive(&sh.q_full);

            const int lim = real ? visible(p, s.r, tok) : s.r.keys;
            const bool busy = warp * 32 < s.n_rows;  // some row of this warp is one
            float m = kNoMax, l = 0.f;
            *reinterpret_cast<uint4 *>(sh.nan_cols[tid]) = make_uint4(0, 0, 0, 0);
            for (int j = tile0; j < tile1; ++j, ++it) {
                if (!(ok = wait_warp(&sh.s_full, it & 1, abort_flag))) break;
                // (complete since before the keys were loaded: the tile's scales)
                if (!(ok = wait_warp(&sh.page_full[it % kAhead], it / kAhead & 1, abort_flag))) break;
                tc_fence_after();
                if (busy) {
                    int page = it % kAhead;  // of the scales
                    float up = row_up;
                    const int seen = lim - j * 128;  // columns of this tile that the row sees
                    const bool edge = j * 128 + 128 > lim_min;
                    uint32_t a[32], b[32];
                    if (edge) {
                        // What the row does not see, as -inf in its scores' place.
#pragma unroll 1
                        for (int x = 0; x < 128; x += 16) {
                            uint32_t r[16];
                            tmem_ld16(lanes + C::kColS + x, r);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (x + i >= seen) r[i] = 0xFF800000u;  // -inf
                            tmem_st16(lanes + C::kColS + x, r);
                        }
                        tmem_wait_st();
                    }
                    float top = -INFINITY;
                    const auto gather = [&](uint32_t (&r)[32], int base) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float2 sc = sh.scale[page][base / 16 + x];
                            top = fmaxf(top, fmaf(max16(r + 16 * x), up * sc.x, sc.y));
                        }
                    };
                    // The maximum first; scores 64..127 stay in registers.
                    tmem_ld32(lanes + C::kColS, a);
                    tmem_ld32(lanes + C::kColS + 32, b);
                    tmem_arrived(a);
                    tmem_arrived(b);
                    gather(a, 0);
                    gather(b, 32);
                    tmem_ld32(lanes + C::kColS + 64, a);
                    tmem_ld32(lanes + C::kColS + 96, b);
                    tmem_arrived(a);
                    tmem_arrived(b);
                    gather(a, 64);
                    gather(b, 96);
                    const bool raise = top - m > kTopExp;
                    float ref = m;  // what comes off the exponents
                    const bool small = sh.small[page] != 0;
                    if (__any_sync(0xffffffffu, raise || fabsf(m) > kExactRef || small)) {
                        top -= kLift<T>;
                        const float half = raise ? exp2_half(m - top) : 1.f, fix = half * half;
                        if (raise) m = top;
                        l = l * half * half;
                        if (j > tile0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll 1
                            for (int x = 0; x < D / 16; ++x) {
                                uint32_t o[16];
                                tmem_ld16(lanes + C::kColO + x * 16, o);
#pragma unroll
                                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
                                tmem_st16(lanes + C::kColO + x * 16, o);
                            }
                        }
                        ref = m;
                        if (__any_sync(0xffffffffu, (fabsf(m) > kExactRef && m != kNoMax) || small)) {
                            // The exponents take the scores' place, and go through the rest as they are.
#pragma unroll 1
                            for (int x = 0; x < 8; ++x) {
                                uint32_t r[16];
                                tmem_ld16(lanes + C::kColS + x * 16, r);
                                const float2 sc = sh.scale[page][x];
                                const float lv = sc.y == -INFINITY ? 0.f : sc.y;
                                float sum = 0.f;
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const float z = fmaf(__uint_as_float(r[i]), up * sc.x, sc.y) - ref;
                                    sum += exp2_fast(z - lv);
                                    r[i] = __float_as_uint(z);
                                }
                                l += sum;
                                tmem_st16(lanes + C::kColS + x * 16, r);
                            }
                            tmem_wait_st();
                            tmem_ld32(lanes + C::kColS + 64, a);
                            tmem_ld32(lanes + C::kColS + 96, b);
                            tmem_arrived(a);
                            tmem_arrived(b);
                            page = kAhead;
                            up = 1.f;
                            ref = 0.f;
                        }
                    }
                    const auto weigh = [&](uint32_t (&r)[32], int base) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float2 sc = sh.scale[page][base / 16 + x];
                            const float2 f = make_float2(up * sc.x, up * sc.x), off = make_float2(sc.y - ref, sc.y - ref);
                            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float2 z = fma2(make_float2(__uint_as_float(r[16 * x + 2 * i]),
                                                                  __uint_as_float(r[16 * x + 2 * i + 1])), f, off);
                                const float2 w = make_float2(exp2_fast(z.x), exp2_fast(z.y));
                                sum.x += w.x, sum.y += w.y;
                                r[8 * x + i] = h2_bits(w.x, w.y);
                            }
                            l = fmaf(sum.x + sum.y, sh.inv_vs[page][base / 16 + x], l);
                        }
                        tmem_st16(lanes + C::kColP + base / 2, r);
                    };
                    weigh(a, 64);
                    tmem_ld32(lanes + C::kColS, a);
                    weigh(b, 96);
                    tmem_ld32(lanes + C::kColS + 32, b);
                    tmem_arrived(a);
                    tmem_arrived(b);
                    weigh(a, 0);
                    weigh(b, 32);
                    tmem_wait_st();
                    if (edge) {
                        // Values with NaN in this tile: the columns of the keys that this row sees.
                        if (!(ok = wait_warp(&sh.v_full, it & 1, abort_flag))) break;
                        if (*static_cast<volatile int *>(&sh.nan[it & 1]) == static_cast<int>(it) + 1) {
                            if (real)
                                mark_nan(p, p.table + s.b * p.table_stride, s.h, j * 128, min(lim, j * 128 + 128),
                                         sh.nan_cols[tid]);
                        }
                    }
                }
                tc_fence_before();
                mbar_arrive(&sh.p_full);
                if (lane == 0) mbar_arrive(&sh.page_empty[it % kAhead]);
            }
            if (!ok || !(ok = wait_warp(&sh.o_full, seg & 1, abort_flag))) break;
            tc_fence_after();
            if (busy) {
                const bool whole = tile0 == 0 && tile1 == s.tiles;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const float lse2 = l == 0.f ? -INFINITY : m + log2f(l);
                const int slot = 2 * blockIdx.x + (tile0 == 0 ? 1 : 0);
                const long long token = s.r.first + tok;
#pragma unroll 1
                for (int x = 0; x < D / 32; ++x) {
                    uint32_t o[32];
                    tmem_ld32(lanes + C::kColO + x * 32, o);
                    tmem_arrived(o);
                    if (!real) continue;
                    const uint32_t bad = sh.nan_cols[tid][x];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float y = __uint_as_float(o[i]) * inv;
                        o[i] = __float_as_uint(bad >> i & 1u ? NAN : y);
                    }
                    if (whole) {
                        T *to = static_cast<T *>(p.o) + token * p.o_st[0] + head * p.o_st[1] + x * 32;
                        if (sa.vec_o) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8) {
                                uint4 w;
                                T *h = reinterpret_cast<T *>(&w);
#pragma unroll
                                for (int k = 0; k < 8; ++k) h[k] = Elem<T>::from_float(__uint_as_float(o[i + k]));
                                *reinterpret_cast<uint4 *>(to + i) = w;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) to[i] = Elem<T>::from_float(__uint_as_float(o[i]));
                        }
                    } else {
                        float *to = sa.part_o + (static_cast<long long>(slot) * kTileRows + tid) * D + x * 32;
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            *reinterpret_cast<uint4 *>(to + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                }
                if (real && whole && p.lse) p.lse[token * p.H + head] = lse2 * 0.6931471805599453f;
                if (real && !whole) sa.part_lse[slot * kTileRows + tid] = lse2;
                // Begun here, ended by a later CTA.
                if (tid == 0 && tile0 == 0 && !whole)
                    sa.desc[blockIdx.x] = StreamDesc{s.last_cta - static_cast<int>(blockIdx.x) + 1, s.r.first, s.h, s.row0, s.n_rows, {}};
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.seg_empty[seg & 1]);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
    if (tid == 0 && *abort_flag && !skip) report_device_error(PMKL_DEVERR_TIMEOUT);
    clear_unused<T>(p);
}

}  // namespace paged
}  // namespace pmkl_b200
