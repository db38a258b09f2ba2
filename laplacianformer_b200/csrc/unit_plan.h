// Which CTA (or CTA pair) of a launch takes which of its work units.
//
// Units go to the P CTAs in turn, long ones (of the problems before the last)
// first: CTA c takes c, c + P and so on.  Where the long units end within a
// turn, the CTAs that got one fewer first take `extra` units of the last
// problem each, about as many as a long one lasts, before the turns go on; with
// a single turn these are the CTAs that got none.  Plain C++ too, so that the
// host can replay a launch.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define LFB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LFB_HOST_DEVICE inline
#endif

namespace lfb {

// The k-th unit of CTA c of P; a number past the last unit: none left.
LFB_HOST_DEVICE int unit_at(int longer, int extra, int c, int P, int k) {
    const int have = longer > c ? (longer - c + P - 1) / P : 0;
    if (k < have) return c + k * P;
    const int j = k - have, ahead = longer % P, behind = P - ahead;
    if (c >= ahead) return j < extra ? longer + j * behind + c - ahead : longer + extra * behind + c + (j - extra) * P;
    return longer + extra * behind + c + j * P;
}

// `extra` for `longer` units, the last of which lasts `ratio` times one of the
// `last` units that follow, on P CTAs.
inline int extra_units(int longer, int last, int P, double ratio) {
    const int ahead = longer % P;
    if (ahead == 0 || last == 0) return 0;
    const int most = last / (P - ahead) + 1;  // more than there are
    return ratio + 0.5 < 2 ? 1 : ratio + 0.5 < most ? (int)(ratio + 0.5) : most;
}

}  // namespace lfb
