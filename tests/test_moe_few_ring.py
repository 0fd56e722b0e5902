"""The ring of FP8 weight stages, on the CPU: csrc/moe_few.h's rule of which group of MMA warps takes which stage, run against
loads that land in any order.

A wait names the parity of a phase.  It returns at once when the slot's barrier is in a phase of the other parity, be that the
phase behind the wanted one or the one before it: a group that has not seen a slot's last phase can pass before its load has landed."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "radeonflow_kernels_b200", "csrc")
CUDA = os.path.dirname(os.path.dirname(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"))

# One CTA: a producer that fills free slots in order, loads that land in an order of the adversary's, two groups that wait by
# parity and free what they took.  Between items group 1 runs ahead of group 0 by one item at most (the exchange of sums).
PROGRAM = r"""
#include "moe_few.h"
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

struct Slot { long done = 0, issued = 0, freed = 0; };   // phases whose load has landed, has been issued, has been freed

// -> false: a group passed a wait for a stage that had not landed
bool run(int stages, unsigned seed, bool slow) {
    std::mt19937 rng(seed);
    std::vector<int> items(200);
    const int fixed = rng() % 3 ? 0 : 1 + rng() % 8;
    for (int& n : items) n = fixed ? fixed : 1 + rng() % 8;
    std::vector<Slot> slot(stages);
    std::vector<long> flight;                 // stages issued and not landed
    long total = 0, issued = 0;
    for (int n : items) total += n;
    struct Group { size_t item = 0; long base = 0; int i = -1; };
    Group g[2];
    for (long step = 0; step < 400 * total; ++step) {
        const int what = rng() % 8;
        if (what == 0) {                      // producer
            if (issued < total && slot[issued % stages].freed == issued / stages) {
                flight.push_back(issued);
                slot[issued % stages].issued++;
                ++issued;
            }
        } else if (what == 1 || (!slow && what < 4)) {          // a load lands
            if (!flight.empty()) {
                const size_t at = slow ? flight.size() - 1 - (rng() % 8 ? 0 : rng() % flight.size()) : rng() % flight.size();
                slot[flight[at] % stages].done++;
                flight.erase(flight.begin() + at);
            }
        } else {
            const int who = what & 1;
            Group& me = g[who];
            if (me.item == items.size()) {
                if (g[1 - who].item == items.size()) return true;
                continue;
            }
            const int n = items[me.item], s = (int)(me.base % stages);
            if (me.i < 0) me.i = rf::few_first_stage(who, s);
            if (me.i >= n) {                  // the item's end: sums are exchanged
                if (who == 0 ? g[1].item <= g[0].item : g[1].item > g[0].item) continue;
                me.base += n;
                ++me.item;
                me.i = -1;
                continue;
            }
            const long stage = me.base + me.i;
            Slot& b = slot[stage % stages];
            const long phase = stage / stages;
            if ((b.done & 1) == (phase & 1)) continue;          // the barrier's phase has the wanted parity: not over yet
            if (b.done != phase + 1) return false;              // passed, and the load had not landed
            b.freed++;
            me.i += 2;
        }
    }
    std::printf("stuck\n");
    return false;
}

int main() {
    int bad = 0;
    for (int ng = 1; ng <= 2; ++ng)
        for (unsigned seed = 0; seed < 400; ++seed) bad += !run(rf::few_stages(true, ng), seed * 2 + ng, seed % 2);
    std::printf("%d\n", bad);
    return bad != 0;
}
"""


@pytest.fixture(scope="module")
def simulate(tmp_path_factory):
    def build(program):
        d = tmp_path_factory.mktemp("ring")
        (d / "ring.cpp").write_text(program)
        subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-I", CSRC, "-I", os.path.join(CUDA, "include"), "-o",
                        str(d / "ring"), str(d / "ring.cpp")], check=True, capture_output=True, text=True)
        return subprocess.run([str(d / "ring")], capture_output=True, text=True, timeout=300)
    return build


def test_no_group_passes_a_stage_that_has_not_landed(simulate):
    out = simulate(PROGRAM)
    assert out.returncode == 0, out.stdout


def test_the_adversary_finds_a_rule_that_lets_one_pass(simulate):
    """Stages in turn by their number inside the item: an odd ring, or an item that starts at an odd slot, changes a slot's group."""
    out = simulate(PROGRAM.replace("rf::few_first_stage(who, s)", "who"))
    assert out.returncode == 1 and int(out.stdout.split()[-1]) > 0 and "stuck" not in out.stdout


def test_the_kernel_uses_the_rule():
    with open(os.path.join(CSRC, "moe_few.cu")) as f:
        s = f.read()
    assert "kStages = few_stages(FP8, NG)" in s and "i = few_first_stage(group, (int)s); i < n_stages; i += 2" in s
