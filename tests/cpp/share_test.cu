// Host test of where the attention kernels' shares begin, for lists of work past
// 32 bits: against the same quotient in 128 bits, and the owner of a tile found
// by the inverse.  Runs no kernel.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <random>

#include "paged_attention_stream.cuh"

using namespace pmkl_b200::paged;

int main() {
    std::mt19937_64 rng(1);
    for (int i = 0; i < 200000; ++i) {
        const long long shares = 1 + static_cast<long long>(rng() % 640);
        long long total = static_cast<long long>(rng() >> (16 + rng() % 40));
        if (i % 5 == 0) total = (1LL << 32) * static_cast<long long>(1 + rng() % 1000);  // whose low half is 0
        if (total < shares) total = shares;
        const long long c = static_cast<long long>(rng() % (shares + 1));
        const long long want = static_cast<long long>(static_cast<unsigned __int128>(total) * c / shares);
        if (share_begin(total, c, shares) != want) {
            std::printf("share %lld of %lld begins at %lld, not %lld\n", c, shares, share_begin(total, c, shares), want);
            return 1;
        }
        // The owner of a tile near the list's beginning, where the product is small, and of any.
        const long long last = i % 2 ? static_cast<long long>(rng() % 1000) % total : static_cast<long long>(rng() % total);
        const long long near = static_cast<long long>(static_cast<unsigned __int128>(shares) * last / total);
        if (share_begin(shares, last, total) != near) {
            std::printf("tile %lld of %lld: owner near %lld, not %lld\n", last, total, share_begin(shares, last, total), near);
            return 1;
        }
    }
    std::printf("shares ok\n");
    return 0;
}
