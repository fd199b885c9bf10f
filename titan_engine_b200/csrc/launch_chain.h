// launch_chain.h — which attention launches may start while those before them still run (programmatic dependent launch).
//
// A kernel of such a chain waits for the launch before it, and so for all before that one, ahead of its first write to what the
// launches share: split-KV rows, arrival counters, outputs.  Until then it reads its layer's pool, q and the new k and v, and writes its
// layer's new rows.  EVERY launch of the chain may still be running at that point (small ones are all resident at once), so none of
// them may be of the same layer, whose new rows it would read or write, or have an output that it reads.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>
#include <vector>

namespace tk {

struct MemRange {
    const void* at;
    size_t bytes;
};

class LaunchChain {
public:
    // A launch of `layer` that reads `in` and writes `out` (empty ranges allowed): may it overlap the launches of the chain?  Either way
    // it is the chain's last one afterwards; one that may not waits for all of them and begins a new chain.
    bool add(bool allowed, int layer, std::initializer_list<MemRange> in, MemRange out) {
        bool overlap = allowed && !links_.empty();
        for (const Link& l : links_) {
            overlap = overlap && l.layer != layer;
            for (const MemRange& r : in) overlap = overlap && !meet(r, l.out);
        }
        if (!overlap) links_.clear();
        links_.push_back({layer, out});
        return overlap;
    }
    void clear() { links_.clear(); }

private:
    struct Link {
        int layer;
        MemRange out;
    };
    static bool meet(const MemRange& a, const MemRange& b) {
        if (!a.at || !b.at || !a.bytes || !b.bytes) return false;
        const uintptr_t x = (uintptr_t)a.at, y = (uintptr_t)b.at;
        return x < y + b.bytes && y < x + a.bytes;
    }
    std::vector<Link> links_;
};

}  // namespace tk
