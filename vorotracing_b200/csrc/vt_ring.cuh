// vt_ring.cuh -- how the roles of a kernel count through its rings of stages, buffers and barriers.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define VT_RING_HD __host__ __device__ __forceinline__
#else
#define VT_RING_HD inline
#endif

namespace vt {
namespace tc {

// Counts through the stages of a ring: index and the parity of its current use.
struct Ring {
    uint32_t i = 0, phase = 0;
    VT_RING_HD void next(uint32_t stages)
    {
        if (++i == stages) { i = 0; phase ^= 1u; }
    }
    VT_RING_HD void skip(uint32_t n, uint32_t stages)  // n at most stages
    {
        i += n;
        if (i >= stages) { i -= stages; phase ^= 1u; }
    }
};

}  // namespace tc

// ---- narrow_kernel (vt_mx8_linear.cu), by dy's columns in chunks of 64 ----

constexpr uint32_t NARROW_SETS = 4;  // of activation warps, which take tiles in turn

// Places of dH in tensor memory, as many as there is room for, up to six
constexpr uint32_t narrow_buffers(uint32_t oc) { return oc == 4 ? 3 : oc == 3 ? 6 : 4; }

// Barriers that tell of a finished dH, in turn.  A parity tells a phase from the one before it, and from the one
// behind it, only if the asker knows that no other is possible.  A set comes to tile j from tile j - 4, so it knows of
// j - 4 and what was before it; and dH of a tile goes no further than its buffer, whose tile j has to leave first.  With a
// barrier for each of three buffers that would be too little: the phase before j's (of tile j - 3) may not have ended,
// or j's may have, while the set was still storing.  Six barriers, whose phase before is tile j - 6's, are enough.
constexpr uint32_t narrow_ready(uint32_t oc) { return narrow_buffers(oc) < NARROW_SETS ? 2u * narrow_buffers(oc) : narrow_buffers(oc); }

}  // namespace vt
