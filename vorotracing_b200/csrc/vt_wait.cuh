// vt_wait.cuh -- how long a kernel has waited, in clocks of its SM.
//
// The clock runs on while the GPU runs another context: one step between two looks at it counts as WAIT_LOOK
// at most (about 2 ms, more than the polls between two looks take), so that a kernel that was set aside does not
// take the others' time for its own.
#pragma once

#ifdef __CUDACC__
#define VT_WAIT_HD __host__ __device__ __forceinline__
#else
#define VT_WAIT_HD inline
#endif

namespace vt {
namespace tc {

constexpr long long WAIT_LIMIT = 2000000000ll;  // about a second
constexpr long long WAIT_LOOK = 1ll << 22;

struct WaitTime {
    long long last, waited;
    VT_WAIT_HD explicit WaitTime(long long now) : last(now), waited(0) {}
    VT_WAIT_HD bool over(long long now)
    {
        const long long step = now - last;
        last = now;
        waited += step < WAIT_LOOK ? step : WAIT_LOOK;
        return waited > WAIT_LIMIT;
    }
};

}  // namespace tc
}  // namespace vt
