"""How a kernel's waits are timed, on the host: a program around csrc/vt_wait.cuh."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include "vt_wait.cuh"
using namespace vt::tc;

// Steps between looks at the clock, `n` of one length: how many until the wait is over, or none
static long long steps(WaitTime &t, long long &now, long long length, long long n)
{
    for (long long i = 1; i <= n; ++i)
        if (t.over(now += length)) return i;
    return 0;
}
int main()
{
    long long now = 1ll << 40;
    WaitTime alone(now);
    std::printf("%lld ", steps(alone, now, 20000, 1000000));  // a wait that nothing interrupts
    WaitTime aside(now);
    std::printf("%lld ", steps(aside, now, 20000, 50000));    // half of its time,
    std::printf("%d ", (int)aside.over(now += 20000000000ll));  // set aside for ten seconds: not its own,
    std::printf("%lld ", steps(aside, now, 20000, 1000000));  // and the rest
    WaitTime slow(now);
    std::printf("%lld\n", steps(slow, now, 1ll << 30, 100000));  // looks far apart: it still ends
}
"""


def test_time_set_aside_is_not_waited(tmp_path):
    src, exe = tmp_path / "wait.cpp", tmp_path / "wait"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-std=c++17", "-I", os.path.join(ROOT, "vorotracing_b200", "csrc"), str(src), "-o", str(exe)])
    limit, look = 2000000000, 1 << 22
    alone, half, aside, rest, slow = map(int, subprocess.check_output([str(exe)], text=True).split())
    assert alone == limit // 20000 + 1 and half == 0
    assert aside == 0
    assert rest == (limit - 50000 * 20000 - look) // 20000 + 1
    assert slow == limit // look + 1
