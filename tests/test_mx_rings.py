"""The roles of narrow_kernel and the barriers between them, played on the host in every order that comes up: the
counts and rings of csrc/vt_ring.cuh, barriers that tell a parity only, as mbarriers do."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
#include "vt_ring.cuh"
using namespace vt;
using tc::Ring;

struct Bar {  // one arrival a phase
    unsigned phase = 0;
    bool over(unsigned parity) const { return (phase & 1u) != parity; }
    void arrive() { ++phase; }
};

// One play: false if no role can go on before all are done, or one finds another tile than its own.
static bool play(uint32_t oc, uint32_t stages, uint32_t tiles, std::mt19937 &rng)
{
    const uint32_t bufs = narrow_buffers(oc), readies = narrow_ready(oc), sets = NARROW_SETS;
    std::vector<Bar> full(stages), empty(stages), dh_full(readies), h_full(bufs);
    std::vector<int> stage(stages, -1), dh(bufs, -1), h(bufs, -1);
    uint32_t copied = 0, first = 0, second = 0, first_done = 0, second_done = 0;  // tiles issued, and products that are over, in order
    Ring cr, fr, fb, fready, fold, sr, sb;
    struct Set { uint32_t tile; Ring r, b, ready; bool stored; } set[8];
    for (uint32_t s = 0; s < sets; ++s) {
        set[s] = {s, {}, {}, {}, true};
        set[s].r.skip(s, stages);
        set[s].b.skip(s, bufs);
        set[s].ready.skip(s, readies);
    }
    std::vector<uint32_t> f_ready, f_buf, s_stage;  // where a product's end arrives
    const uint32_t roles = 5 + sets;
    std::vector<uint32_t> slow(roles);
    for (auto &x : slow) x = rng() % 4 ? 1 : 1 + rng() % 200;  // some roles are asked rarely
    bool mixed = false;
    const auto step = [&](uint32_t who) {  // whether that role could go on
        if (who == 0 && copied < tiles && empty[cr.i].over(cr.phase ^ 1u)) {  // copies
            stage[cr.i] = (int)copied++;
            full[cr.i].arrive();
            cr.next(stages);
            return true;
        }
        if (who == 1 && first < tiles && full[fr.i].over(fr.phase) && (first < bufs || empty[fold.i].over(fold.phase))) {  // dH
            mixed |= stage[fr.i] != (int)first;
            if (first >= bufs) fold.next(stages);
            f_ready.push_back(fready.i);
            f_buf.push_back(fb.i);
            ++first;
            fr.next(stages);
            fb.next(bufs);
            fready.next(readies);
            return true;
        }
        if (who == 2 && first_done < first) {  // the end of one
            dh[f_buf[first_done]] = (int)first_done;
            dh_full[f_ready[first_done]].arrive();
            ++first_done;
            return true;
        }
        if (who == 3 && second < tiles && h_full[sb.i].over(sb.phase) && full[sr.i].over(sr.phase)) {  // dW
            mixed |= h[sb.i] != (int)second || stage[sr.i] != (int)second;
            s_stage.push_back(sr.i);
            ++second;
            sr.next(stages);
            sb.next(bufs);
            return true;
        }
        if (who == 4 && second_done < second) {
            empty[s_stage[second_done]].arrive();
            ++second_done;
            return true;
        }
        if (who < 5) return false;
        Set &x = set[who - 5];  // activations: take a tile, and then its stores
        if (!x.stored) {
            x.stored = true;
            x.tile += sets;
            x.r.skip(4, stages);
            x.b.skip(bufs < 4u ? bufs : 4u, bufs);
            if (bufs < 4u) x.b.skip(4u - bufs, bufs);
            x.ready.skip(4, readies);
            return true;
        }
        if (x.tile < tiles && full[x.r.i].over(x.r.phase) && dh_full[x.ready.i].over(x.ready.phase)) {
            mixed |= stage[x.r.i] != (int)x.tile || dh[x.b.i] != (int)x.tile;
            h[x.b.i] = (int)x.tile;
            h_full[x.b.i].arrive();
            x.stored = false;
            return true;
        }
        return false;
    };
    uint32_t idle = 0;
    while (second_done < tiles && !mixed) {
        const uint32_t who = rng() % roles;
        if (rng() % slow[who] == 0 && step(who)) idle = 0;
        else if (++idle > 500) {
            bool any = false;
            for (uint32_t w = 0; w < roles; ++w) any |= step((who + w) % roles);
            if (!any) return false;
            idle = 0;
        }
    }
    return !mixed;
}
int main(int, char **argv)
{
    const uint32_t oc = atoi(argv[1]), stages = atoi(argv[2]);
    std::mt19937 rng(oc * 100 + stages);
    for (int i = 0; i < 3000; ++i)
        if (!play(oc, stages, 1 + rng() % 60, rng)) {
            std::printf("play %d stands still or mixes tiles up\n", i);
            return 1;
        }
    return 0;
}
"""


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    d = tmp_path_factory.mktemp("rings")
    (d / "rings.cpp").write_text(PROGRAM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "vorotracing_b200", "csrc"), str(d / "rings.cpp"), "-o", str(d / "rings")])
    return str(d / "rings")


@pytest.mark.parametrize("oc,stages", [(1, 5), (1, 12), (2, 5), (2, 8), (3, 7), (3, 12), (4, 4), (4, 5), (4, 10), (4, 12)])
def test_no_order_stands_still(exe, oc, stages):
    r = subprocess.run([exe, str(oc), str(stages)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
