"""The tiles that attention through a window goes through (windlass_amd/csrc/window.h), checked on the host against what
every node sees: no device."""
import subprocess

import pytest

from windlass_amd import build

SOURCE = r"""
#include <cstdio>
#include "window.h"
using namespace wl::paged;
int main() {
    const unsigned windows[] = {1, 2, 5, 16, 31, 32, 33, 47, 64, 65, 100, 160, 0x7FFFFFFFu}, all_sinks[] = {0, 1, 4, 31, 32, 33, 70, 0x7FFFFFFFu};
    const unsigned all_nodes[] = {1, 2, 3, 8, 17, 32, 33, 64};
    const unsigned part = PART;  // keys that a kernel masks at a time, in tiles of 32
    unsigned lost = 0, open = 0, late = 0, tiles = 0;
    for (unsigned window : windows) for (unsigned sinks : all_sinks) for (unsigned nodes : all_nodes) for (unsigned len = 0; len < 330; len++) {
        const Skip skip = window_skip(len, window, sinks, 32);
        const unsigned last = (len + nodes + 31) / 32;  // tiles of all keys
        for (unsigned depth = 0; depth < nodes; depth++) {
            const unsigned pos = len + depth;
            auto sees = [&](unsigned k) { return k < len && (k < sinks || (unsigned long long)k + window > pos); };
            for (unsigned k = 0; k < len; k++)
                if (skip.at != ~0u && k / 32 >= skip.at && k / 32 < skip.at + skip.n && sees(k)) lost++;
            if (window_from(pos, window) < len && !sees(window_from(pos, window))) lost++;
            if (window_from(pos, window) > 0 && window_from(pos, window) - 1 < len && window_from(pos, window) - 1 >= sinks && sees(window_from(pos, window) - 1)) lost++;
            bool before[64] = {};  // in walks from a tile on: whether a part before this one had a key that the node sees
            for (unsigned t = 0; t < last; t++) {
                if (t >= skip.at && t < skip.at + skip.n) continue;
                for (unsigned k0 = 32 * t; k0 < 32 * t + 32; k0 += part) {
                    if (k0 >= len) continue;
                    unsigned n = 0;
                    for (unsigned k = k0; k < k0 + part; k++) n += sees(k);
                    const bool masked = k0 + part > len || window_masks(len, nodes, window, sinks, k0, part);
                    tiles++;
                    if (!masked && n != part) open++;
                    for (unsigned s = 0; s <= t; s++)  // a walk that begins with tile s
                        if (n && !before[s]) {
                            before[s] = true;
                            if (k0 != 32 * s && !masked && !(s >= skip.at && s < skip.at + skip.n)) late++;
                        }
                }
            }
        }
    }
    std::printf("%u tiles: seen and left out %u, unseen and not masked %u, first seen and not masked %u\n", tiles, lost, open, late);
    return lost || open || late;
}
"""


@pytest.mark.parametrize("part", [32, 16])
def test_tiles_of_a_window(tmp_path, part):
    """No key that a node sees is left out; what some node does not see is masked; and in a walk from any tile on, the
    first keys that a node sees are in the walk's first tile or in a masked one (where its reference is set)."""
    src = tmp_path / "w.cpp"
    src.write_text(SOURCE.replace("PART", str(part)))
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", build.CSRC, str(src), "-o", str(tmp_path / "w")], check=True)
    r = subprocess.run([str(tmp_path / "w")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout.split()[0]) > 10 ** 6
