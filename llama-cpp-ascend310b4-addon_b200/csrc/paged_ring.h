// paged_ring.h -- the copies of paged_prefill_kernel's ring in order, and what is
// left of them when a wait has run out.  Plain arithmetic, tested without a device.
#pragma once

#include <stdint.h>

#include "args.h"

namespace b200 {

// Barriers of one kind, passed round robin (a ring's stages; one barrier is a ring of
// one): `counts` phases were entered by the two copying warps, each with arrivals of
// its own.  Neither enters a barrier's next phase before the last one has completed,
// so they are at most a lap apart.
struct PfPhases {
    uint32_t counts[2];
    uint32_t stages;
    B200_HD uint32_t most() const { return counts[0] > counts[1] ? counts[0] : counts[1]; }
    B200_HD uint32_t least() const { return counts[0] < counts[1] ? counts[0] : counts[1]; }
    // (the arrivals of one warp are missing in the phases least() .. most() - 1)
    // the phases whose copies may be in flight: the last of every barrier
    B200_HD uint32_t oldest() const { return most() > stages ? most() - stages : 0; }
    B200_HD uint32_t stage(uint32_t phase) const { return phase % stages; }
    B200_HD uint32_t parity(uint32_t phase) const { return (phase / stages) & 1u; }
};

// Waits for the copies of barriers that were left behind: the arrivals of the warp that
// stopped first are made up for, then every barrier's last phase is waited for.
template <class Arrive, class Wait>
B200_HD inline void pf_land_phases(const PfPhases& p, Arrive arrive, Wait wait) {
    for (uint32_t i = p.least(); i < p.most(); ++i) arrive(p.stage(i));
    for (uint32_t i = p.oldest(); i < p.most(); ++i) wait(p.stage(i), p.parity(i));
}

}  // namespace b200
