// A ring of NS stages in shared memory: which stage a fill lies in, which phase of that stage's barrier it completes, and
// which fills may still be in flight.  Plain C++, so that the rule is tested on the host.
#pragma once

#ifdef __CUDACC__
#define B200Q_HD __host__ __device__ __forceinline__
#else
#define B200Q_HD inline
#endif

namespace b200q {

// A wait at the end has to be for a stage's last fill and no other.  It is made by parity: for the fill before, it returns while
// the last is in flight and blocks once that has landed; so does one for a fill that was never made, the other way round.
template <int NS>
struct Ring {
    static B200Q_HD int stage(int fill) { return fill % NS; }
    static B200Q_HD unsigned parity(int fill) { return (unsigned)(fill / NS) & 1u; }
    // after fills 0 .. issued - 1: those from here on are their stages' last
    static B200Q_HD int oldest(int issued) { return issued > NS ? issued - NS : 0; }
    // the last fill of the stage of `fill`, the newest that could have been made (below 0: none)
    static B200Q_HD int last(int fill, bool made) { return made ? fill : fill - NS; }
};

}  // namespace b200q
