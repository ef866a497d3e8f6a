"""What the kernels' synchronisation relies on, checked on the CPU: no run on a GPU shows a missing wait reliably."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "lookatmyquant_b200" / "csrc"


def test_a_warp_reconverges_before_an_aligned_cluster_barrier():
    """barrier.cluster with .aligned needs all threads of a warp at the instruction. The attention kernels' first warp comes
    to it from a branch of one lane: each such instruction has a __syncwarp() before it in its function."""
    found = 0
    for src in sorted(CSRC.glob("*.cu*")):
        text = src.read_text()
        for m in re.finditer(r"barrier\.cluster\.arrive[a-z.]*\.aligned", text):
            body = text[text.rindex("{\n", 0, m.start()):m.start()]
            assert "__syncwarp();" in body, src.name
            found += 1
    assert found


STEPS = r"""
#include <cstdio>
#include <vector>
#include "attention_steps.cuh"
using namespace lamq;

// What the issuing thread commits, in its order: (barrier, the last step of each query tile whose P it had waited for by
// then). A warp's program: its waits, each after the P of `after` steps of its tile.
struct Commit { int bar, seen[2]; };

template <int NB>
int check(int n0, int n1, bool by_buffer) {
    const Steps<NB> s{n0, n1};
    std::vector<Commit> done;
    int seen[2] = {0, 0};
    for (int u = 0; u < NB && u < s.count(); ++u) done.push_back({u, {0, 0}});
    for (int u = 0; u < s.count(); ++u) {
        ++seen[s.query_tile(u)];
        if (u == s.ends_first()) done.push_back({NB, {seen[0], seen[1]}});
        done.push_back({u % NB, {seen[0], seen[1]}});
    }
    const auto ok = [&](Wait w, int t, int after) {  // completes without this tile's later arrivals, the next one does not
        int c = 0;
        for (const Commit &e : done) {
            if (e.bar != w.bar) continue;
            if (c == w.phase && e.seen[t] > after) return false;
            if (c == w.phase + 1 && e.seen[t] <= after) return false;
            ++c;
        }
        return c > w.phase;
    };
    int bad = 0;
    for (int t = 0; t < 2; ++t) {
        const int n = t ? n1 : n0;
        for (int j = 0; j < n; ++j) {
            if (s.query_tile(s.index(j, t)) != t) ++bad;
            if (!ok(s.scores(s.index(j, t)), t, j)) ++bad;
            if (j > 0 && !ok(s.read(s.index(j - 1, t)), t, j)) ++bad;
        }
        if (n > 0) {
            const int last = s.index(n - 1, t);
            if (!ok(by_buffer ? s.read(last) : s.last_read(last), t, n)) ++bad;
        }
    }
    return bad;
}

int main() {
    int bad = 0, by_buffer = 0;
    for (int n0 = 0; n0 < 12; ++n0)
        for (int n1 = 0; n1 < 12; ++n1) {
            bad += check<2>(n0, n1, false) + check<3>(n0, n1, false);
            by_buffer += check<2>(n0, n1, true);
        }
    std::printf("%d %d\n", bad, by_buffer);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no C++ compiler")
def test_no_wait_of_the_attention_forward_can_miss_its_phase(tmp_path):
    """An mbarrier wait tests a parity: a barrier that completes a second time before a slow warp has looked makes it wait
    for good. For every number of key tiles, each wait's completion comes without an arrival that the warp makes later,
    and the next completion of that barrier needs one. (With a tile's last step read off its buffer's barrier, as a plant,
    the check finds steps of the other tile that complete it again.)"""
    src, exe = tmp_path / "steps.cpp", tmp_path / "steps"
    src.write_text(STEPS)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{CSRC}", "-x", "c++", str(src), "-o", str(exe)], check=True)
    bad, by_buffer = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert bad == 0 and by_buffer > 0


def test_skinny_updates_keep_the_cut_of_their_long_sums():
    """A = X·Xᵀ of a skinny matrix is a few tiles of long sums: they are cut into pieces over the idle SMs, whose fp32 sums the
    workspace holds, for a batch of two and for the longest as for one."""
    from lookatmyquant_b200 import _lib
    from lookatmyquant_b200.build import LIB, build
    if not LIB.exists():
        build()
    size, tile = _lib.load().lamq_newton_schulz_workspace_size, 128 * 128 * 4
    up = lambda v, to: -(-v // to) * to
    plain = lambda b, m, n: 4 * up(b * m * up(n, 64) * 2, 256) + 4 * up(b * min(m, n) * up(min(m, n), 64) * 2, 256)
    for b, m, n, tiles in ((1, 16, 9728, 1), (2, 16, 9728, 2), (1, 64, 131072, 1), (1, 512, 9728, 16), (2, 9728, 256, 8)):
        assert size(b, m, n) >= plain(b, m, n) + tiles * tile * min(148 // tiles, up(max(m, n), 64) // 64 // 4), (b, m, n)
    for b, m, n in ((1, 2560, 9728), (4, 960, 2560), (1, 2560, 2560)):  # enough tiles: whole sums
        assert size(b, m, n) < plain(b, m, n) + tile
