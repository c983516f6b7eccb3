// Entries that the threads of a launch take (launch_index.h), for launches of up to 2^32 - 1 threads: each of the array's once, and none outside it.  Prints "ok", or the first that is not
// as it should be (exit status 1).
#include <algorithm>
#include <cstdio>
#include <vector>

#include "../../spy_amd/csrc/launch_index.h"

int main() {
    const uint32_t threads = 1024;
    for (uint32_t blocks : {1u, 2u, 7u, 1025u, (1u << 20) + 1000u, (1u << 21) - 1u, 1u << 21, 2u * ((1u << 20) + 1000u), (1u << 22) - 1u})
        for (int n : {1, 3, 1023, 1024, 1025, 5000, (1 << 20) - 1}) {
            std::vector<int> taken(n, 0);
            for (uint32_t block = 0; block < blocks; block++) {
                if (block == 2048 && blocks > 4096) block = std::max(block, blocks / 2 - 1024);         // the first ones, those around the middle, and the last
                if (block == blocks / 2 + 1024 && blocks > 8192) block = blocks - 2048;
                for (uint32_t thread = 0; thread < threads; thread++)
                    for (int64_t i = launch_first(block, threads, thread); i < n; i += launch_step(blocks, threads)) {
                        if (i < 0) { std::printf("%u blocks, %d entries: block %u, thread %u takes %lld\n", blocks, n, block, thread, (long long)i); return 1; }
                        taken[i]++;
                    }
            }
            for (int i = 0; i < n; i++)
                if (taken[i] != 1) { std::printf("%u blocks: entry %d of %d taken %d times\n", blocks, i, n, taken[i]); return 1; }
        }
    std::puts("ok");
}
