// The rings' rule (csrc/ring.cuh) for the host: which fills the attention kernels wait for before a block ends, and a stage's
// barrier, whose phases complete one after another as fills land and whose wait for a parity returns unless the phase that is
// running has it.
#include "ring.cuh"

#include <vector>

using b200q::Ring;

// Fills 0 .. base - 1 were made, and of the next `more` those in mask.  waits: the fills waited for.  Returns 0 if each stage that
// has a fill is waited for exactly once, by a wait that blocks while its last fill is in flight and returns once that has
// landed; else 1 + a stage.
template <int NS>
static int check(int base, int more, int mask, const std::vector<int>& waits) {
    std::vector<int> fills(NS, 0), met(NS, 0);
    for (int i = 0; i < base + more; i++)
        if (i < base || mask >> (i - base) & 1) fills[Ring<NS>::stage(i)]++;
    for (int w : waits) {
        const int st = Ring<NS>::stage(w), phases = fills[st];
        if (phases == 0) return 1 + st;
        auto returns = [&](int complete) { return (unsigned)(complete & 1) != Ring<NS>::parity(w); };
        if (returns(phases - 1) || !returns(phases)) return 1 + st;
        met[st]++;
    }
    for (int st = 0; st < NS; st++)
        if (met[st] != (fills[st] > 0)) return 1 + st;
    return 0;
}

// as the loaders wait after `issued` fills without a gap
template <int NS>
static int plain(int issued) {
    std::vector<int> waits;
    for (int i = Ring<NS>::oldest(issued); i < issued; i++) waits.push_back(i);
    return check<NS>(issued, 0, 0, waits);
}
// as the row kernel's producer waits after a batch of eight of which some were made
template <int NS>
static int gap(int base, int mask) {
    std::vector<int> waits;
    for (int i = base + 8 > NS ? base + 8 - NS : 0; i < base; i++) waits.push_back(i);
    for (int l = 0; l < 8; l++) {
        const int mine = Ring<NS>::last(base + l, mask >> l & 1);
        if (mine >= 0) waits.push_back(mine);
    }
    return check<NS>(base, 8, mask, waits);
}

extern "C" int ring_plain(int stages, int issued) {
    return stages == 2 ? plain<2>(issued) : stages == 4 ? plain<4>(issued) : stages == 24 ? plain<24>(issued) : stages == 48 ? plain<48>(issued) : -1;
}
extern "C" int ring_gap(int stages, int base, int mask) { return stages == 24 ? gap<24>(base, mask) : stages == 48 ? gap<48>(base, mask) : -1; }
