// most_splits of split_share.h: shares of a launch's pages in 32 bits, as the kernels compute them, against the quotient in 64 bits.
#include <algorithm>
#include <cstdio>

#include "split_share.h"

int main() {
    const uint64_t pages_of[] = {1, 2, 15, 125, 2048, 65537, 1 << 20, (1 << 23) - 1, 1 << 23, (1 << 24) - 4097, (1 << 24) - 1, 1 << 24,
                                 (1 << 24) + 5, (1 << 25) + 1, (1 << 26) - 1, 1 << 26};
    for (uint64_t pages : pages_of) {
        for (uint64_t asked : {1, 2, 63, 64, 255, 256, 300, 511, 512, 65536}) {
            const unsigned splits = (unsigned)std::min<uint64_t>(asked, skv::most_splits(pages));
            if (splits < std::min<uint64_t>(asked, 63) || (pages < (1 << 23) - 4096 && asked <= 512 && splits != asked)) return 1;
            for (unsigned span : {(unsigned)pages, (unsigned)pages + 4096u})
                for (unsigned split = 0; split <= splits; ++split)
                    if ((split * span) / splits != (uint64_t)split * span / splits) {
                        std::printf("split %u of %u of %u pages\n", split, splits, span);
                        return 1;
                    }
        }
    }
    std::printf("ok\n");
    return 0;
}
