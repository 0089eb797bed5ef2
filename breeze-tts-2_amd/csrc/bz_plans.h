// Launch shapes chosen by a fitted cost, kept for each host thread: choosing one
// takes 0.5 (bz_mx_gemm) or 0.7 us (bz_gemm_tiled), and a call asks twice, for
// its workspace and for its launch.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cstring>

namespace bz {

// What a plan follows from.
struct PlanKey {
    int32_t type, M, N, K, cfg;
    bool operator==(const PlanKey& o) const { return std::memcmp(this, &o, sizeof o) == 0; }
};

// Plan of `key` from make(plan), which returns a status; the last plan of each
// of 64 places is kept, and only good ones.
template <class Plan, class Make>
int planned(const PlanKey& key, Plan& plan, Make&& make) {
    struct Entry {
        PlanKey key;
        Plan plan;
    };
    static thread_local Entry kept[64] = {};  // (no plan has M = 0)
    uint32_t h = 0;
    for (uint32_t v : {(uint32_t)key.type, (uint32_t)key.M, (uint32_t)key.N, (uint32_t)key.K, (uint32_t)key.cfg})
        h = (h ^ v) * 0x9E3779B1u;
    Entry& e = kept[h >> 26];
    if (!(e.key == key)) {
        const int rc = make(plan);
        if (rc != 0) return rc;
        e.key = key;
        e.plan = plan;
    }
    plan = e.plan;
    return 0;
}

}  // namespace bz
