// Rows cut into runs, a launch each, where their items of eight values do not
// fit the 32 bits a launch counts them in.  Host code without HIP.
#pragma once

#include <algorithm>
#include <cstdint>

namespace bz {

// Rows of K columns that one launch takes: at most 2^31 items.
inline int rows_per_launch(int M, int K) { return (int)std::min<int64_t>(M, ((int64_t)1 << 31) / (K / 8)); }

// run(first row, rows) for each of them until one returns something else than
// 0; that is the answer.  The count goes on past the last run's start, so it
// has 64 bits: with runs of 2^29 rows (K = 32) the fourth ends at 2^31.
template <class Run>
int for_row_runs(int M, int K, Run&& run) {
    const int rows = rows_per_launch(M, K);
    for (int64_t m0 = 0; m0 < M; m0 += rows) {
        const int rc = run(m0, (int)std::min<int64_t>(rows, M - m0));
        if (rc != 0) return rc;
    }
    return 0;
}

}  // namespace bz
