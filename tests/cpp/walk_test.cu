// Host test of the walk through the attention kernels' shared-out work: over
// random batches every tile of every item belongs to exactly one CTA, an item's
// CTAs follow one another, and the CTA that begins an item knows the one that
// ends it.  Runs no kernel.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "paged_attention_stream.cuh"

using namespace pmkl_b200::paged;

template <int ROWS, int KEYS, int COST>
bool check(std::mt19937 &rng, int grid) {
    auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
    const int batch = pick(1, 9), group = pick(1, 5), kv = pick(1, 3), block = 16, width = pick(1, 40);
    std::vector<int> lens(batch), starts(batch + 1, 0);
    for (int b = 0; b < batch; ++b) {
        lens[b] = pick(0, 3) ? pick(0, width * block) : pick(0, 3);
        starts[b + 1] = starts[b] + (pick(0, 4) ? pick(0, 60) : pick(0, 1));
    }
    AttnArgs p{};
    p.seq_lens = lens.data();
    p.query_starts = starts.data();
    p.tokens = starts[batch];
    p.batch = batch;
    p.H = kv * group;
    p.Hkv = kv;
    p.block = block;
    p.max_blocks = width;
    p.max_q = 60;
    p.causal = pick(0, 1);
    std::vector<long long> end(batch);
    long long total = 0;
    std::vector<std::vector<int>> seen;  // of every (b, h, row tile): the CTA of each tile
    std::vector<long long> first(batch + 1, 0);
    for (int b = 0; b < batch; ++b) {
        const Request r = request_of(p, b);
        total += head_tiles<ROWS, KEYS, COST>(p, r, group) * kv;
        end[b] = total;
        for (int h = 0; h < kv; ++h)
            for (int row0 = 0; row0 < r.rows * group; row0 += ROWS)
                seen.emplace_back(tile_count<ROWS, KEYS, COST>(p, r, row0, r.rows * group, group), -1);
        first[b + 1] = static_cast<long long>(seen.size());
    }
    std::vector<std::pair<int, int>> ends;  // (item, the CTA that its first CTA says ends it)
    const long long shares = std::min<long long>(total, grid);
    for (int c = 0; c < shares; ++c) {
        Share w{};
        w.total = total;
        w.shares = shares;
        w.u = share_begin(total, c, shares);
        w.u_end = share_begin(total, c + 1, shares);
        while (end[w.b] <= w.u) ++w.b;
        w.b_begin = w.b ? end[w.b - 1] : 0;
        Segment s;
        int guard = 0;
        while (next_segment<ROWS, KEYS, COST>(p, w, s)) {
            if (++guard > 100000) return std::printf("no end\n"), false;
            const Request r = request_of(p, s.b);
            const int n_rt = (r.rows * group + ROWS - 1) / ROWS;
            if (s.row0 % ROWS || s.row0 >= r.rows * group || s.h >= kv) return std::printf("no such item\n"), false;
            const long long item = first[s.b] + static_cast<long long>(s.h) * n_rt + s.row0 / ROWS;
            std::vector<int> &t = seen[item];
            if (s.tiles != static_cast<int>(t.size()) || s.tile0 >= s.tile1 || s.tile1 > s.tiles)
                return std::printf("tiles %d..%d of %d\n", s.tile0, s.tile1, s.tiles), false;
            if (s.n_rows != std::min(ROWS, r.rows * group - s.row0)) return std::printf("rows\n"), false;
            for (int i = s.tile0; i < s.tile1; ++i) {
                if (t[i] >= 0) return std::printf("a tile twice\n"), false;
                t[i] = c;
            }
            if (s.tile0 == 0 && s.tile1 < s.tiles) ends.emplace_back(static_cast<int>(item), s.last_cta);
        }
    }
    for (const auto &t : seen)
        for (size_t i = 0; i < t.size(); ++i)
            if (t[i] < 0 || (i && t[i] != t[i - 1] && t[i] != t[i - 1] + 1)) return std::printf("a tile left out\n"), false;
    for (const auto &e : ends)
        if (seen[e.first].back() != e.second) return std::printf("wrong last CTA\n"), false;
    return true;
}

int main() {
    std::mt19937 rng(1);
    for (int i = 0; i < 4000; ++i) {
        const int grid = std::uniform_int_distribution<int>(1, i % 3 ? 20 : 320)(rng);
        if (!check<8, 128, 3>(rng, grid) || !check<16, 192, 3>(rng, grid) || !check<32, 128, 3>(rng, grid) ||
            !check<128, 128, 1>(rng, grid)) {
            std::printf("FAILED at %d\n", i);
            return 1;
        }
    }
    std::printf("walk ok\n");
    return 0;
}
