// How the tensors of one call of the norm are shared out over launches.
#pragma once
#include <algorithm>
#include <vector>

namespace lb {

struct NormPass {
    int from, to;      // tensors
    long long chunks;  // of all of them
    int keep;          // the last ones, left in the L2 for the second pass
};

// `chunks[k]`: those of tensor k (an empty one has none, and takes no place). At most `most` tensors with elements a pass. The second pass walks all of them
// backwards, so that the last `keep` chunks of the whole call are what it meets first.
inline std::vector<NormPass> norm_passes(const std::vector<long long>& chunks, int most, int keep) {
    std::vector<NormPass> passes;
    const int n = (int)chunks.size();
    for (int k = 0; k < n;) {
        NormPass p{k, k, 0, 0};
        for (int held = 0; k < n && held < most; k++) held += chunks[k] > 0, p.chunks += chunks[k];
        p.to = k;
        passes.push_back(p);
    }
    for (size_t k = passes.size(); k-- > 0;) {
        passes[k].keep = (int)std::min<long long>(keep, passes[k].chunks);
        keep -= passes[k].keep;
    }
    return passes;
}

}  // namespace lb
