// Walking a count in batches (host only, no CUDA).
#pragma once
#include <algorithm>

namespace vdb {

// 0 .. total - 1 in batches of `size` and a last one of what is left. `at` passes the last
// batch by up to `size`, which a 32-bit total next to 2^31 has no room for.
struct Batches {
    int total, size;
    long long at = 0;

    // The next batch: first .. first + n - 1; false after the last one.
    bool next(int& first, int& n) {
        if (at >= total) return false;
        first = (int)at;
        n = (int)std::min<long long>(size, total - at);
        at += size;
        return true;
    }
};

}  // namespace vdb
